"""Thin host wrappers: torch ROCm tensors are used only as device buffers; every op below is one
call into libty1.so (hand-written gfx950 kernels) on the current torch stream."""
import ctypes
import functools
import operator
from array import array

import torch

from . import _lib

DENSE_K_ALIGN = 32


def _chk(t, dtype, name):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f'{name}: expected a tensor on the GPU (ROCm device)')
    if t.dtype != dtype:
        raise TypeError(f'{name}: expected {dtype}, got {t.dtype}')
    if not t.is_contiguous():
        raise ValueError(f'{name}: must be contiguous')
    return t


def _chk_out(t, dtype, shape, name):
    """A caller-provided output buffer: its raw pointer goes to a kernel, so type, device, layout and shape must fit."""
    _chk(t, dtype, name)
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f'{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}')
    return t


def round_up(v, m):
    return (v + m - 1) // m * m


def fold_bn(gamma, beta, mean, var, eps=1e-3):
    """NumPy (host) in/out: scale, shift of an inference BatchNormalization (Keras eps 1e-3)."""
    import numpy as np
    g, b, m, v = (np.ascontiguousarray(a, np.float32) for a in (gamma, beta, mean, var))
    scale = np.empty_like(g)
    shift = np.empty_like(g)
    _lib.call('ty1_fold_bn', g.ctypes.data, b.ctypes.data, m.ctypes.data, v.ctypes.data,
              float(eps), int(g.shape[0]), scale.ctypes.data, shift.ctypes.data)
    return scale, shift


def conv3x3_workspace_bytes(N, H, W, Cin, Cout, pool):
    """Scratch bytes ty1_conv3x3_bn_leaky_ws_f32 wants for this problem (0: it would not split its tail)."""
    import ctypes
    n = ctypes.c_size_t(0)
    _lib.call('ty1_conv3x3_workspace_bytes', N, H, W, Cin, Cout, int(bool(pool)), ctypes.addressof(n))
    return int(n.value)


def conv3x3_bn_leaky(x, w_ohwi, scale, shift, pool, alpha=0.1, out=None, workspace=None):
    """x (N,H,W,Cin) NHWC f32 -> (N,H/2,W/2,Cout) if pool else (N,H,W,Cout).
    workspace: optional 1-D uint8/float32 device tensor used as scratch for the K-split tail."""
    _chk(x, torch.float32, 'x'); _chk(w_ohwi, torch.float32, 'w')
    _chk(scale, torch.float32, 'scale'); _chk(shift, torch.float32, 'shift')
    N, H, W, Cin = x.shape
    Cout = w_ohwi.shape[0]
    assert tuple(w_ohwi.shape) == (Cout, 3, 3, Cin), w_ohwi.shape
    oshape = (N, H // 2, W // 2, Cout) if pool else (N, H, W, Cout)
    if out is None:
        out = torch.empty(oshape, dtype=torch.float32, device=x.device)
    else:
        _chk(out, torch.float32, 'out')
        assert tuple(out.shape) == oshape
    if workspace is None:
        _lib.call('ty1_conv3x3_bn_leaky_f32', x.data_ptr(), w_ohwi.data_ptr(), scale.data_ptr(), shift.data_ptr(),
                  out.data_ptr(), N, H, W, Cin, Cout, int(bool(pool)), float(alpha), _lib.current_stream())
    else:
        if not workspace.is_cuda or not workspace.is_contiguous():
            raise ValueError('workspace must be a contiguous tensor on the GPU')
        _lib.call('ty1_conv3x3_bn_leaky_ws_f32', x.data_ptr(), w_ohwi.data_ptr(), scale.data_ptr(), shift.data_ptr(),
                  out.data_ptr(), N, H, W, Cin, Cout, int(bool(pool)), float(alpha), workspace.data_ptr(),
                  workspace.numel() * workspace.element_size(), _lib.current_stream())
    return out


def static_scratch_bytes():
    return int(_lib.lib().ty1_static_scratch_bytes())


def static_scratch_init():
    """Resolve the static scratch array's address on the current device (once per device, outside graph capture)."""
    _lib.call('ty1_static_scratch_init')


def set_reserved_cus(k):
    """Persistent grids leave k CUs free from now on (0: fill the chip).  Results do not depend on k."""
    _lib.call('ty1_set_reserved_cus', int(k))


def get_reserved_cus():
    import ctypes
    k = ctypes.c_int(0)
    _lib.call('ty1_get_reserved_cus', ctypes.byref(k))
    return int(k.value)


def conv3x3_bn_leaky_static(x, w_ohwi, scale, shift, pool, alpha, out):
    """The conv block through the entry point that allocates nothing (ty1_conv3x3_bn_leaky_static_f32): the caller
    brings every buffer, the K-split scratch is the library's static device array."""
    _chk(x, torch.float32, 'x'); _chk(w_ohwi, torch.float32, 'w')
    _chk(scale, torch.float32, 'scale'); _chk(shift, torch.float32, 'shift')
    N, H, W, Cin = x.shape
    Cout = w_ohwi.shape[0]
    assert tuple(w_ohwi.shape) == (Cout, 3, 3, Cin), w_ohwi.shape
    _chk_out(out, torch.float32, (N, H // 2, W // 2, Cout) if pool else (N, H, W, Cout), 'out')
    _lib.call('ty1_conv3x3_bn_leaky_static_f32', x.data_ptr(), w_ohwi.data_ptr(), scale.data_ptr(), shift.data_ptr(),
              out.data_ptr(), N, H, W, Cin, Cout, int(bool(pool)), float(alpha), _lib.current_stream())
    return out


def conv3x3_workspace_bytes_bf16(N, H, W, Cin, Cout, pool):
    """Scratch bytes ty1_conv3x3_bn_leaky_bf16 wants for this problem."""
    import ctypes
    n = ctypes.c_size_t(0)
    _lib.call('ty1_conv3x3_workspace_bytes_bf16', N, H, W, Cin, Cout, int(bool(pool)), ctypes.addressof(n))
    return int(n.value)


def cast_bf16(x, out=None):
    """f32 device tensor -> bf16 (round to nearest even) with the library's own kernel."""
    _chk(x, torch.float32, 'x')
    if out is None:
        out = torch.empty(x.shape, dtype=torch.bfloat16, device=x.device)
    else:
        _chk(out, torch.bfloat16, 'out')
        assert out.shape == x.shape
    _lib.call('ty1_cast_f32_to_bf16', x.data_ptr(), out.data_ptr(), x.numel(), _lib.current_stream())
    return out


def conv3x3_bn_leaky_bf16(x, w_ohwi, scale, shift, pool, alpha=0.1, out_f32=False, out=None, workspace=None):
    """The conv block of the bf16 network.  Cin == 3: x and w are f32 (first layer), otherwise bf16; the result is
    bf16, or f32 with out_f32 (unpooled layers only).  fp32 accumulation and epilogue."""
    N, H, W, Cin = x.shape
    in_dt = torch.float32 if Cin == 3 else torch.bfloat16
    _chk(x, in_dt, 'x'); _chk(w_ohwi, in_dt, 'w')
    _chk(scale, torch.float32, 'scale'); _chk(shift, torch.float32, 'shift')
    Cout = w_ohwi.shape[0]
    assert tuple(w_ohwi.shape) == (Cout, 3, 3, Cin), w_ohwi.shape
    oshape = (N, H // 2, W // 2, Cout) if pool else (N, H, W, Cout)
    out_dt = torch.float32 if out_f32 else torch.bfloat16
    if out is None:
        out = torch.empty(oshape, dtype=out_dt, device=x.device)
    else:
        _chk(out, out_dt, 'out')
        assert tuple(out.shape) == oshape
    if workspace is not None and (not workspace.is_cuda or not workspace.is_contiguous()):
        raise ValueError('workspace must be a contiguous tensor on the GPU')
    _lib.call('ty1_conv3x3_bn_leaky_bf16', x.data_ptr(), w_ohwi.data_ptr(), scale.data_ptr(), shift.data_ptr(),
              out.data_ptr(), N, H, W, Cin, Cout, int(bool(pool)), float(alpha), int(bool(out_f32)),
              workspace.data_ptr() if workspace is not None else None,
              workspace.numel() * workspace.element_size() if workspace is not None else 0, _lib.current_stream())
    return out


def conv3x3_x2_c3_bf16(x, w0, scale0, shift0, w1, scale1, shift1, alpha=0.1, out=None):
    """The first two conv blocks of the bf16 network in ONE launch (ty1_conv3x3_x2_c3_bf16): x (N,H,W,3) f32, w0 (16,3,3,3)
    f32, w1 (32,3,3,16) bf16 -> (N,H/4,W/4,32) bf16; the 16-channel tensor between the blocks stays in LDS."""
    _chk(x, torch.float32, 'x'); _chk(w0, torch.float32, 'w0'); _chk(w1, torch.bfloat16, 'w1')
    for name, t in (('scale0', scale0), ('shift0', shift0), ('scale1', scale1), ('shift1', shift1)):
        _chk(t, torch.float32, name)
    N, H, W, cin = x.shape
    if cin != 3 or tuple(w0.shape) != (16, 3, 3, 3) or tuple(w1.shape) != (32, 3, 3, 16):
        raise ValueError(f'conv3x3_x2_c3_bf16: x {tuple(x.shape)}, w0 {tuple(w0.shape)}, w1 {tuple(w1.shape)} are not the 3 -> 16 -> 32 blocks')
    if scale0.numel() != 16 or shift0.numel() != 16 or scale1.numel() != 32 or shift1.numel() != 32:
        raise ValueError('conv3x3_x2_c3_bf16: scale / shift sizes must be 16 and 32')
    oshape = (N, H // 4, W // 4, 32)
    if out is None:
        out = torch.empty(oshape, dtype=torch.bfloat16, device=x.device)
    else:
        _chk_out(out, torch.bfloat16, oshape, 'out')
    _lib.call('ty1_conv3x3_x2_c3_bf16', x.data_ptr(), w0.data_ptr(), scale0.data_ptr(), shift0.data_ptr(), w1.data_ptr(),
              scale1.data_ptr(), shift1.data_ptr(), out.data_ptr(), N, H, W, float(alpha), _lib.current_stream())
    return out


def preprocess_u8(img_u8, out_hw=(448, 448), swap_rb=False, out=None):
    """uint8 (H0,W0,3) image on the device -> fp32 (out_h,out_w,3) in [0,1]: cv2.resize INTER_LINEAR + /255
    (utils.py:11-15).  `out` may be one slot x[n] of the network's input batch."""
    _chk(img_u8, torch.uint8, 'img')
    H0, W0, c = img_u8.shape
    assert c == 3
    if out is None:
        out = torch.empty((out_hw[0], out_hw[1], 3), dtype=torch.float32, device=img_u8.device)
    else:
        _chk(out, torch.float32, 'out')
        assert tuple(out.shape) == (out_hw[0], out_hw[1], 3)
    _lib.call('ty1_preprocess_u8', img_u8.data_ptr(), H0, W0, int(bool(swap_rb)), out.data_ptr(), out_hw[0], out_hw[1],
              _lib.current_stream())
    return out


def preprocess_batch_u8(imgs_u8, out_hw=(448, 448), swap_rb=False, out=None):
    """uint8 (n,H0,W0,3) equal-sized frames on the device -> fp32 (n,out_h,out_w,3) in [0,1] in ONE launch; frame by frame
    the bits of preprocess_u8 (utils.py:11-15 over the batch loop of data_sequence.py:94-99, or over a camera's frames)."""
    _chk(imgs_u8, torch.uint8, 'imgs')
    if imgs_u8.dim() != 4 or imgs_u8.shape[3] != 3:
        raise ValueError(f'imgs: expected (n,H0,W0,3) uint8, got {tuple(imgs_u8.shape)}')
    n, H0, W0, _ = imgs_u8.shape
    shape = (n, out_hw[0], out_hw[1], 3)
    out = torch.empty(shape, dtype=torch.float32, device=imgs_u8.device) if out is None else _chk_out(out, torch.float32, shape, 'out')
    _lib.call('ty1_preprocess_batch_u8', imgs_u8.data_ptr(), n, H0, W0, int(bool(swap_rb)), out.data_ptr(), out_hw[0], out_hw[1],
              _lib.current_stream())
    return out


def pick_splits(K, n_rows, units, slots=None, chunk=DENSE_K_ALIGN):
    """Split-K factor for the Dense GEMM: the number of blocks (tiles * splits) that best fills ONE round of `slots`
    resident blocks, with at least 4 chunks (32 floats / 64 bf16 of K) per slice.  slots: 2 per CU for the 64 x 64 tiles
    of batches above 32, 1 per CU for the 32 x 128 tiles below (every extra split is one more partial for the kernel
    behind the GEMM to reduce: measured with tools/experiments/dense_splits.py, GEMM + tail at 32 images 52 -> 34 us
    with 21 splits instead of 85, at one image 49 -> 40 us)."""
    chunks = K // chunk
    tiles = ((n_rows + 63) // 64) * ((units + 63) // 64) if n_rows > 32 else (units + 127) // 128
    if slots is None:
        slots = 512 if n_rows > 32 else 256
    best, best_eff = 1, 0.0
    for s in range(1, max(1, chunks // 4) + 1):
        blocks = tiles * s
        if blocks > slots:
            break
        eff = blocks / (-(-blocks // slots) * slots)
        if eff > best_eff + 1e-9:
            best, best_eff = s, eff
    return best


def dense_splitk(x, wt, units, splits=None, part=None):
    """x (N,K), wt (rows>=units, ldk) transposed Dense weight, both f32 or both bf16 -> f32 partials (splits,N,ldz)."""
    bf = x.dtype == torch.bfloat16
    _chk(x, torch.bfloat16 if bf else torch.float32, 'x'); _chk(wt, x.dtype, 'wt')
    N, K = x.shape
    ldk = wt.shape[1]
    if splits is None:
        splits = pick_splits(K, N, units, chunk=64 if bf else DENSE_K_ALIGN)
    ldz = round_up(units, 4)
    if part is None:
        part = torch.empty((splits, N, ldz), dtype=torch.float32, device=x.device)
    else:
        _chk(part, torch.float32, 'part')
        if part.dim() != 3 or part.shape[1] != N or part.shape[2] < units:
            raise ValueError(f'part: expected (splits, {N}, >= {units}), got {tuple(part.shape)}')
        splits, _, ldz = part.shape
    if wt.shape[0] < units or ldk < K:
        raise ValueError(f'wt: expected (>= {units}, >= {K}), got {tuple(wt.shape)}')
    _lib.call('ty1_dense_splitk_bf16' if bf else 'ty1_dense_splitk_f32', x.data_ptr(), wt.data_ptr(), part.data_ptr(), N, K, units, ldk, ldz,
              splits, _lib.current_stream())
    return part


def head_activate(part, bias, S=7, B=2, C=20, out=None):
    """partials (splits,N,ldz) [+ bias (units)] -> y (N,S,S,C+5B) = [softmax C | sigmoid B | sigmoid 4B]."""
    _chk(part, torch.float32, 'part')
    if part.dim() == 2:
        part = part.unsqueeze(0)
    splits, N, ldz = part.shape
    if bias is not None:
        _chk(bias, torch.float32, 'bias')
        if bias.numel() < S * S * (C + 5 * B):
            raise ValueError(f'bias: expected {S * S * (C + 5 * B)} values, got {bias.numel()}')
    if ldz < S * S * (C + 5 * B):
        raise ValueError(f'part: last dimension {ldz} is smaller than the {S * S * (C + 5 * B)} Dense units')
    if out is None:
        out = torch.empty((N, S, S, C + 5 * B), dtype=torch.float32, device=part.device)
    else:
        _chk_out(out, torch.float32, (N, S, S, C + 5 * B), 'out')
    _lib.call('ty1_head_activate_f32', part.data_ptr(), _lib.ptr(bias), out.data_ptr(), N, S, B, C, ldz, splits,
              _lib.current_stream())
    return out


def decode_nms(pred, B=2, C=20, img_size=448, iou_thr=0.2, out=None):
    """pred (N,S,S,C+5B) f32 -> boxes (N,S*S*B,4) f64, score (N,S*S*B) f32, cls i32, keep u8."""
    _chk(pred, torch.float32, 'pred')
    if pred.dim() == 3:
        pred = pred.unsqueeze(0)
    N, S = pred.shape[0], pred.shape[1]
    if pred.shape[2] != S or pred.shape[3] != C + 5 * B:
        raise ValueError(f'pred shape {tuple(pred.shape)} does not match S,S,C+5B with B={B}, C={C}')
    slots = S * S * B
    if out is None:
        dev = pred.device
        out = (torch.empty((N, slots, 4), dtype=torch.float64, device=dev),
               torch.empty((N, slots), dtype=torch.float32, device=dev),
               torch.empty((N, slots), dtype=torch.int32, device=dev),
               torch.empty((N, slots), dtype=torch.uint8, device=dev))
    boxes, score, cls, keep = out
    _chk_out(boxes, torch.float64, (N, slots, 4), 'boxes'); _chk_out(score, torch.float32, (N, slots), 'score')
    _chk_out(cls, torch.int32, (N, slots), 'cls'); _chk_out(keep, torch.uint8, (N, slots), 'keep')
    _lib.call('ty1_decode_nms', pred.data_ptr(), N, S, B, C, int(img_size), float(iou_thr),
              boxes.data_ptr(), score.data_ptr(), cls.data_ptr(), keep.data_ptr(), _lib.current_stream())
    return boxes, score, cls, keep


def head_decode_nms(part, bias, S=7, B=2, C=20, img_size=448, iou_thr=0.2, y=None, out=None):
    """Dense partials (splits,N,ldz) [+ bias] -> detections in ONE launch (head_activate + decode_nms, same bits).
    y: optional (N,S,S,C+5B) f32 tensor that also receives the head tensor."""
    _chk(part, torch.float32, 'part')
    if part.dim() == 2:
        part = part.unsqueeze(0)
    splits, N, ldz = part.shape
    units, slots = S * S * (C + 5 * B), S * S * B
    if ldz < units:
        raise ValueError(f'part: last dimension {ldz} is smaller than the {units} Dense units')
    if bias is not None:
        _chk(bias, torch.float32, 'bias')
        if bias.numel() < units:
            raise ValueError(f'bias: expected {units} values, got {bias.numel()}')
    if y is not None:
        _chk_out(y, torch.float32, (N, S, S, C + 5 * B), 'y')
    if out is None:
        dev = part.device
        out = (torch.empty((N, slots, 4), dtype=torch.float64, device=dev), torch.empty((N, slots), dtype=torch.float32, device=dev),
               torch.empty((N, slots), dtype=torch.int32, device=dev), torch.empty((N, slots), dtype=torch.uint8, device=dev))
    boxes, score, cls, keep = out
    _chk_out(boxes, torch.float64, (N, slots, 4), 'boxes'); _chk_out(score, torch.float32, (N, slots), 'score')
    _chk_out(cls, torch.int32, (N, slots), 'cls'); _chk_out(keep, torch.uint8, (N, slots), 'keep')
    _lib.call('ty1_head_decode_nms_f32', part.data_ptr(), _lib.ptr(bias), _lib.ptr(y), N, S, B, C, ldz, splits, int(img_size),
              float(iou_thr), boxes.data_ptr(), score.data_ptr(), cls.data_ptr(), keep.data_ptr(), _lib.current_stream())
    return boxes, score, cls, keep


def pack_detections(boxes, score, cls, keep, out=None):
    """-> (N, slots, 6) f64 records x0,y0,x1,y1,score,class (-1 where not kept): the unit of the detection gather."""
    _chk(boxes, torch.float64, 'boxes'); _chk(score, torch.float32, 'score'); _chk(cls, torch.int32, 'cls'); _chk(keep, torch.uint8, 'keep')
    N, slots = score.shape
    for name, t, shp in (('boxes', boxes, (N, slots, 4)), ('cls', cls, (N, slots)), ('keep', keep, (N, slots))):
        if tuple(t.shape) != shp:
            raise ValueError(f'{name}: expected shape {shp}, got {tuple(t.shape)}')
    if out is None:
        out = torch.empty((N, slots, 6), dtype=torch.float64, device=boxes.device)
    else:
        _chk_out(out, torch.float64, (N, slots, 6), 'out')
    _lib.call('ty1_pack_detections', boxes.data_ptr(), score.data_ptr(), cls.data_ptr(), keep.data_ptr(), out.data_ptr(),
              N * slots, _lib.current_stream())
    return out


def yolo_head(feats, img_size=448):
    _chk(feats, torch.float32, 'feats')
    if feats.dim() != 5 or feats.shape[-1] != 4 or feats.shape[1] != feats.shape[2]:
        raise ValueError(f'feats must be (N,S,S,B,4), got {tuple(feats.shape)}')
    N, S, _, B, _ = feats.shape
    xy = torch.empty((N, S, S, B, 2), dtype=torch.float32, device=feats.device)
    wh = torch.empty_like(xy)
    _lib.call('ty1_yolo_head_f32', feats.data_ptr(), xy.data_ptr(), wh.data_ptr(), N, S, B, int(img_size),
              _lib.current_stream())
    return xy, wh


def iou(pred_mins, pred_maxes, true_mins, true_maxes):
    shape = torch.broadcast_shapes(pred_mins.shape, pred_maxes.shape, true_mins.shape, true_maxes.shape)
    ops = [_chk(t.expand(shape).contiguous(), torch.float32, 'iou operand')
           for t in (pred_mins, pred_maxes, true_mins, true_maxes)]
    if shape[-1] != 2:
        raise ValueError('last axis must be (x, y)')
    out = torch.empty(shape[:-1], dtype=torch.float32, device=ops[0].device)
    _lib.call('ty1_iou_f32', *(o.data_ptr() for o in ops), out.data_ptr(), out.numel(), _lib.current_stream())
    return out


def yolo_head_np(feats, img_size=448):
    """NumPy twin: feats (...,S,S,B,4) f32 -> xy float64, wh float32 (tiny_yolov1.py:36-55)."""
    _chk(feats, torch.float32, 'feats')
    shape = feats.shape
    S, B = shape[-3], shape[-2]
    if shape[-1] != 4 or shape[-4] != S:
        raise ValueError(f'feats must be (...,S,S,B,4), got {tuple(shape)}')
    N = feats.numel() // (S * S * B * 4)
    xy = torch.empty(shape[:-1] + (2,), dtype=torch.float64, device=feats.device)
    wh = torch.empty(shape[:-1] + (2,), dtype=torch.float32, device=feats.device)
    _lib.call('ty1_yolo_head_np_f64', feats.data_ptr(), xy.data_ptr(), wh.data_ptr(), N, S, B, int(img_size),
              _lib.current_stream())
    return xy, wh


def iou_f64(pred_mins, pred_maxes, true_mins, true_maxes):
    shape = torch.broadcast_shapes(pred_mins.shape, pred_maxes.shape, true_mins.shape, true_maxes.shape)
    ops_ = [_chk(t.to(torch.float64).expand(shape).contiguous(), torch.float64, 'iou operand')
            for t in (pred_mins, pred_maxes, true_mins, true_maxes)]
    out = torch.empty(shape[:-1], dtype=torch.float64, device=ops_[0].device)
    _lib.call('ty1_iou_f64', *(o.data_ptr() for o in ops_), out.data_ptr(), out.numel(), _lib.current_stream())
    return out


def yolo_loss_fwd_bwd(y_true, y_pred, B=2, C=20, img_size=448, want_grad=True, loss_out=None):
    """-> loss (1,) f32 batch SUM, loss_per_image (N,), grad (N,S,S,C+5B) or None.
    loss_out: optional (1,) f32 device tensor the batch loss is written to (e.g. a slot of the gradient bucket)."""
    _chk(y_true, torch.float32, 'y_true'); _chk(y_pred, torch.float32, 'y_pred')
    N, S = y_pred.shape[0], y_pred.shape[1]
    if tuple(y_true.shape) != (N, S, S, C + 5) or tuple(y_pred.shape) != (N, S, S, C + 5 * B):
        raise ValueError(f'shapes {tuple(y_true.shape)} / {tuple(y_pred.shape)} do not match B={B}, C={C}')
    dev = y_pred.device
    per = torch.empty((max(N, 1),), dtype=torch.float32, device=dev)
    loss = torch.empty((1,), dtype=torch.float32, device=dev) if loss_out is None else _chk_out(loss_out, torch.float32, (1,), 'loss_out')
    grad = torch.empty_like(y_pred) if want_grad else None
    _lib.call('ty1_yolo_loss_fwd_bwd', y_true.data_ptr(), y_pred.data_ptr(), N, S, B, C, int(img_size),
              per.data_ptr(), loss.data_ptr(), _lib.ptr(grad), _lib.current_stream())
    return loss, per[:N], grad


def train_tail(part, bias, y_true, ldz, S=7, B=2, C=20, img_size=448, y=None, dz=None, loss_out=None):
    """Dense partials (splits,N,ldz_part) [+ bias], labels (N,S,S,C+5) -> loss (1,) batch SUM, loss_per_image (N,), dz (N,ldz)
    in ONE launch + the batch sum (head_activate + yolo_loss_fwd_bwd + head_activate_bwd, same bits).
    y: optional (N,S,S,C+5B) tensor that also receives the head tensor; loss_out: optional (1,) slot for the loss."""
    _chk(part, torch.float32, 'part'); _chk(y_true, torch.float32, 'y_true')
    if part.dim() == 2:
        part = part.unsqueeze(0)
    splits, N, ldz_part = part.shape
    units = S * S * (C + 5 * B)
    if ldz_part < units or ldz < units:
        raise ValueError(f'train_tail: leading dimensions {ldz_part} / {ldz} are smaller than the {units} Dense units')
    if tuple(y_true.shape) != (N, S, S, C + 5):
        raise ValueError(f'y_true {tuple(y_true.shape)} does not match N={N}, S={S}, C={C}')
    if bias is not None:
        _chk(bias, torch.float32, 'bias')
        if bias.numel() < units:
            raise ValueError(f'bias: expected {units} values, got {bias.numel()}')
    if y is not None:
        _chk_out(y, torch.float32, (N, S, S, C + 5 * B), 'y')
    dev = part.device
    dz = torch.empty((N, ldz), dtype=torch.float32, device=dev) if dz is None else _chk_out(dz, torch.float32, (N, ldz), 'dz')
    per = torch.empty((max(N, 1),), dtype=torch.float32, device=dev)
    loss = torch.empty((1,), dtype=torch.float32, device=dev) if loss_out is None else _chk_out(loss_out, torch.float32, (1,), 'loss_out')
    _lib.call('ty1_train_tail_f32', part.data_ptr(), _lib.ptr(bias), y_true.data_ptr(), _lib.ptr(y), dz.data_ptr(), N, S, B, C,
              ldz_part, splits, int(img_size), ldz, per.data_ptr(), loss.data_ptr(), _lib.current_stream())
    return loss, per[:N], dz


def head_activate_bwd(y, grad_y, ldz, B=2, C=20, out=None):
    _chk(y, torch.float32, 'y'); _chk(grad_y, torch.float32, 'grad_y')
    N, S = y.shape[0], y.shape[1]
    if tuple(grad_y.shape) != tuple(y.shape) or y.shape[-1] != C + 5 * B or ldz < y[0].numel():
        raise ValueError(f'head_activate_bwd: y {tuple(y.shape)}, grad_y {tuple(grad_y.shape)}, ldz {ldz} do not fit B={B}, C={C}')
    if out is None:
        out = torch.empty((N, ldz), dtype=torch.float32, device=y.device)
    else:
        _chk_out(out, torch.float32, (N, ldz), 'out')
    _lib.call('ty1_head_activate_bwd_f32', y.data_ptr(), grad_y.data_ptr(), out.data_ptr(), N, S, B, C, ldz,
              _lib.current_stream())
    return out


def dense_wgrad(dz, x, units, dwt, db):
    _chk(dz, torch.float32, 'dz'); _chk(x, torch.float32, 'x'); _chk(dwt, torch.float32, 'dwt'); _chk(db, torch.float32, 'db')
    N, K = x.shape
    if dz.shape[0] != N or dz.shape[1] < units or dwt.shape[0] < units or dwt.shape[1] < K or db.numel() < units:
        raise ValueError(f'dense_wgrad: dz {tuple(dz.shape)}, x {tuple(x.shape)}, dwt {tuple(dwt.shape)}, db {tuple(db.shape)} '
                         f'do not fit units={units}')
    _lib.call('ty1_dense_wgrad_f32', dz.data_ptr(), x.data_ptr(), dwt.data_ptr(), db.data_ptr(), N, K, units,
              dwt.shape[1], dz.shape[1], _lib.current_stream())
    return dwt, db


def adam_step(p, g, m, v, t, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-7):
    for name, a in (('p', p), ('g', g), ('m', m), ('v', v)):
        _chk(a, torch.float32, name)
    _lib.call('ty1_adam_step_f32', p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(), p.numel(),
              float(lr), float(beta1), float(beta2), float(eps), int(t), _lib.current_stream())


# ------------------------------------------------------------------ low-rank adapters, gradient clipping
MAX_RANK, MAX_ADAPTERS = 128, 4096          # of ty1_adapter_*


# the handle of a device's current stream: the call behind torch.cuda.current_stream(i).cuda_stream without the Stream object (1 us)
_stream_of = getattr(torch._C, '_cuda_getCurrentRawStream', None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call_on(index, name, *args):
    """The call on device `index` and its current torch stream: the tensors' device, whatever the current one is."""
    if index != torch.cuda.current_device():
        with torch.cuda.device(index):
            return _lib.call(name, *args, _stream_of(index))
    return _lib.call(name, *args, _stream_of(index))


@functools.lru_cache(maxsize=256)
def _adapter_workspace_bytes(N, K, U, L, R, backward):
    size = ctypes.c_size_t(0)
    _lib.call('ty1_adapter_workspace_bytes', N, K, U, L, R, backward, ctypes.addressof(size))
    return size.value


def _strided(t, dtype, shape, index, name):
    """A tensor on device `index` with a dense last axis and any strides in front of it."""
    if not isinstance(t, torch.Tensor) or t.get_device() != index:
        raise TypeError(f'{name}: expected a tensor on GPU {index}')
    if t.dtype != dtype:
        raise TypeError(f'{name}: expected {dtype}, got {t.dtype}')
    if t.shape != shape:
        raise ValueError(f'{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}')
    if shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f'{name}: the last axis must be dense, its stride is {t.stride(-1)}')
    return t


def _dense_on(t, shape, index, name):
    """A contiguous float32 tensor of this shape on device `index`."""
    _strided(t, torch.float32, shape, index, name)
    if not t.is_contiguous():
        raise ValueError(f'{name}: must be contiguous')
    return t


def _span(t):
    """First and last address + 1 of a tensor's values."""
    lo = t.data_ptr()
    return lo, lo + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size() if t.numel() else lo


def _chk_written(outs, ins):
    """Outputs that the caller brings: rows that do not overlap one another, and memory apart from the operands'."""
    for name, t in outs:
        st, n = t.stride(), t.shape
        need = n[-1]
        for d in range(t.dim() - 2, -1, -1):
            if n[d] > 1 and st[d] < need:
                raise ValueError(f'{name}: strides {st} make its rows overlap')
            need = st[d] * (n[d] - 1) + need
    spans = [(name, *_span(t)) for name, t in list(outs) + list(ins)]
    for i in range(len(outs)):
        for j in range(i + 1, len(spans)):
            if spans[i][1] < spans[j][2] and spans[j][1] < spans[i][2]:
                raise ValueError(f'{spans[i][0]}: shares memory with {spans[j][0]}')


def _adapter_operands(x, a, b, index, scale):
    """Checks the operands both passes share -> (device index, N, K, U, L, R)."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise TypeError('x: expected a tensor on the GPU (ROCm device)')
    if x.dtype is not torch.float32 and x.dtype is not torch.bfloat16:
        raise TypeError(f'x: expected torch.float32 or torch.bfloat16, got {x.dtype}')
    for name, t in (('a', a), ('b', b), ('index', index), ('scale', scale)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f'{name}: expected a tensor on the GPU, got {type(t).__name__}')
    if x.dim() != 2 or a.dim() != 3 or b.dim() != 3:
        raise ValueError(f'expected x (N,K), a (L,R,K), b (L,R,U), got {tuple(x.shape)}, {tuple(a.shape)}, {tuple(b.shape)}')
    dev = x.get_device()
    N, K = x.shape
    L, R, U = b.shape
    if not (1 <= R <= MAX_RANK and 1 <= L <= MAX_ADAPTERS):
        raise ValueError(f'{L} adapters of rank {R}: 1 to {MAX_ADAPTERS} of rank 1 to {MAX_RANK} are supported')
    if K < 1 or U < 1 or max(N, K, U) > 2 ** 30:
        raise ValueError(f'x (N,K) = {(N, K)}, b (L,R,U) = {(L, R, U)}: sizes must be positive (N may be 0) and at most 2^30')
    if (a.dtype is x.dtype and b.dtype is x.dtype and a.get_device() == dev and b.get_device() == dev and a.shape == (L, R, K)
            and index.dtype is torch.int32 and index.get_device() == dev and index.shape == (N,) and index.is_contiguous()
            and scale.dtype is torch.float32 and scale.get_device() == dev and scale.shape == (L,) and scale.is_contiguous()
            and x.stride(1) == 1 and a.stride(2) == 1 and b.stride(2) == 1):
        return dev, N, K, U, L, R                       # the common case; what does not fit is named below, or fits after all
    _strided(x, x.dtype, (N, K), dev, 'x'); _strided(a, x.dtype, (L, R, K), dev, 'a'); _strided(b, x.dtype, (L, R, U), dev, 'b')
    _strided(index, torch.int32, (N,), dev, 'index'); _strided(scale, torch.float32, (L,), dev, 'scale')
    return dev, N, K, U, L, R


def adapter_forward(x, a, b, index, scale, out=None, accumulate=False, h=None):
    """The low-rank adapters of many requests in one batch, beside the Dense layer that they share:
        out[n] = scale[i] * (x[n] . a[i]^T) . b[i],   i = index[n]
    x (N,K), a (L,R,K), b (L,R,U): all float32 or all bfloat16, last axis dense, any strides in front of it (a row of x may be
    repeated by expand); index (N) int32; scale (L) float32 -> out (N,U) float32, sums in float32.
    index[n] < 0: no adapter for this row (zeros).  index[n] >= L: the row becomes NaN (the index lives on the GPU and is not
    read by the host).  Smaller ranks: zero rows in a and b.
    out: where to write.  accumulate: add to what out holds instead (rows without an adapter stay as they are), e.g. to
    part[-1][:, :U], the last of dense_splitk's partials: whatever kernel reduces those then adds the adapters on the way.
    h: optional (N,R) float32 that receives x . a^T (without scale) for adapter_backward."""
    dev, N, K, U, L, R = _adapter_operands(x, a, b, index, scale)
    if out is None:
        if accumulate:
            raise ValueError('accumulate needs out')
        out = torch.empty((N, U), dtype=torch.float32, device=x.device)
        if h is not None:
            _chk_written([('h', _dense_on(h, (N, R), dev, 'h'))], [('x', x), ('a', a), ('b', b), ('index', index), ('scale', scale)])
    else:
        outs = [('out', _strided(out, torch.float32, (N, U), dev, 'out'))]
        if h is not None:
            outs.append(('h', _dense_on(h, (N, R), dev, 'h')))
        _chk_written(outs, [('x', x), ('a', a), ('b', b), ('index', index), ('scale', scale)])
    if N == 0:
        return out
    ws = torch.empty((_adapter_workspace_bytes(N, K, U, L, R, 0),), dtype=torch.uint8, device=x.device)
    _call_on(dev, 'ty1_adapter_forward_bf16' if x.dtype is torch.bfloat16 else 'ty1_adapter_forward_f32', x.data_ptr(), a.data_ptr(),
             b.data_ptr(), index.data_ptr(), scale.data_ptr(), out.data_ptr(), _lib.ptr(h), N, K, U, L, R, x.stride(0), a.stride(1),
             a.stride(0), b.stride(1), b.stride(0), out.stride(0), int(bool(accumulate)), ws.data_ptr(), ws.numel())
    return out


def adapter_backward(dz, x, a, b, index, scale, h=None, want_dx=False, da=None, db=None, dx=None):
    """Gradients of adapter_forward from dz (N,U) float32 = dL/dout -> (da (L,R,K), db (L,R,U), dx (N,K) or None), float32.
    h: what adapter_forward stored, or None: computed again.  da, db, dx: optional buffers; they are written whole (zeros for
    an adapter without rows, for a dx row without an adapter; NaN for the dx row of an index >= L).  want_dx: also the
    gradient of x (the detector's backbone is frozen and needs none); giving dx asks for it too.
    The rows of an adapter are summed in a fixed order: the same bits every time."""
    dev, N, K, U, L, R = _adapter_operands(x, a, b, index, scale)
    _strided(dz, torch.float32, (N, U), dev, 'dz')
    if h is not None:
        _dense_on(h, (N, R), dev, 'h')
    if da is not None or db is not None or dx is not None:
        given = [(name, _strided(t, torch.float32, shape, dev, name)) for name, t, shape in
                 (('da', da, (L, R, K)), ('db', db, (L, R, U)), ('dx', dx, (N, K))) if t is not None]
        _chk_written(given, [('dz', dz), ('x', x), ('a', a), ('b', b), ('index', index), ('scale', scale)] + ([('h', h)] if h is not None else []))
    da = torch.empty((L, R, K), dtype=torch.float32, device=x.device) if da is None else da
    db = torch.empty((L, R, U), dtype=torch.float32, device=x.device) if db is None else db
    if dx is None and want_dx:
        dx = torch.empty((N, K), dtype=torch.float32, device=x.device)
    ws = torch.empty((_adapter_workspace_bytes(N, K, U, L, R, 1),), dtype=torch.uint8, device=x.device)
    _call_on(dev, 'ty1_adapter_backward_bf16' if x.dtype is torch.bfloat16 else 'ty1_adapter_backward_f32', dz.data_ptr(), x.data_ptr(),
             a.data_ptr(), b.data_ptr(), index.data_ptr(), scale.data_ptr(), _lib.ptr(h), da.data_ptr(), db.data_ptr(), _lib.ptr(dx),
             N, K, U, L, R, dz.stride(0), x.stride(0), a.stride(1), a.stride(0), b.stride(1), b.stride(0), da.stride(1), da.stride(0),
             db.stride(1), db.stride(0), dx.stride(0) if dx is not None else 0, ws.data_ptr(), ws.numel())
    return da, db, dx


_DTYPE = operator.attrgetter('dtype')


def _tensor_lists(**lists):
    """One tensor or equally long lists of contiguous tensors on one GPU, float32 or bfloat16, with as many values list by list ->
    (device index, n, the lists' addresses, value counts, types): the HOST arrays of ty1_grad_norm and its kin, as array.array
    (keep them until the call)."""
    T, first, out = torch.Tensor, None, []
    for name, ts in lists.items():
        ts = [ts] if isinstance(ts, T) else list(ts)
        for kind in {*map(type, ts)}:
            if not issubclass(kind, T):
                raise TypeError(f'{name}: expected tensors, got {kind.__name__}')
        if first is None:
            if not ts:
                raise ValueError(f'{name}: no tensors')
            first, n, dev, dtypes, counts = name, len(ts), ts[0].get_device(), [*map(_DTYPE, ts)], [*map(T.numel, ts)]
            if dev < 0:
                raise TypeError(f'{name}: expected tensors on the GPU (ROCm device)')
            for dt in {*dtypes}:
                if dt is not torch.float32 and dt is not torch.bfloat16:
                    raise TypeError(f'{name}: expected torch.float32 or torch.bfloat16, got {dt}')
        else:
            if len(ts) != n:
                raise ValueError(f'{name}: {len(ts)} tensors, {first} has {n}')
            if [*map(_DTYPE, ts)] != dtypes:
                raise TypeError(f'{name}: expected tensors of the types of {first}')
            if [*map(T.numel, ts)] != counts:
                bad = next(k for k, t in enumerate(ts) if t.numel() != counts[k])
                raise ValueError(f'{name}: tensor {bad} has {ts[bad].numel()} values, in {first} it has {counts[bad]}')
        if {*map(T.get_device, ts)} != {dev}:
            raise TypeError(f'{name}: all tensors must be on GPU {dev}')
        if not all(map(T.is_contiguous, ts)):
            raise ValueError(f'{name}: must be contiguous')
        out.append(array('Q', map(T.data_ptr, ts)))
    kinds = array('i', [dt is torch.bfloat16 for dt in dtypes]) if torch.bfloat16 in dtypes else None
    return dev, n, out, array('q', counts), kinds


def _at(a):
    return None if a is None else a.buffer_info()[0]


@functools.lru_cache(maxsize=256)
def _norm_workspace_bytes(n):
    size = ctypes.c_size_t(0)
    _lib.call('ty1_grad_norm_workspace_bytes', n, ctypes.addressof(size))
    return size.value


def _norm_buffers(dev, n, norm):
    device = torch.device('cuda', dev)
    ws = torch.empty((_norm_workspace_bytes(n),), dtype=torch.uint8, device=device)
    return ws, torch.empty((1,), dtype=torch.float32, device=device) if norm is None else _dense_on(norm, (1,), dev, 'norm')


def _max_norm(v):
    v = float(v)
    if not v > 0.0:
        raise ValueError(f'max_norm must be positive, got {v}')
    return v


def grad_norm(grads, norm=None):
    """The global 2-norm of one tensor or a list of tensors (float32 or bfloat16, contiguous, any sizes) -> (1,) float32 on
    the device: squares and sums in float64, in an order fixed by the sizes.  norm: optional (1,) buffer."""
    dev, n, (g,), counts, kinds = _tensor_lists(grads=grads)
    ws, norm = _norm_buffers(dev, n, norm)
    _call_on(dev, 'ty1_grad_norm', _at(g), _at(counts), _at(kinds), n, norm.data_ptr(), ws.data_ptr(), ws.numel())
    return norm


def clip_grad_norm(grads, max_norm, out=None, norm=None):
    """Scales one tensor or a list of tensors by min(1, max_norm / global norm), in place or into out (as many tensors of the
    same numbers of values and types) -> the norm before clipping, (1,) float32 on the device.  A norm that is not finite makes every
    value NaN (Keras' global_clipnorm, tf.clip_by_global_norm).  Tensors must not overlap one another."""
    max_norm = _max_norm(max_norm)
    dev, n, arrays, counts, kinds = _tensor_lists(grads=grads, out=out) if out is not None else _tensor_lists(grads=grads)
    ws, norm = _norm_buffers(dev, n, norm)
    _call_on(dev, 'ty1_clip_grad_norm', _at(arrays[0]), _at(arrays[-1]), _at(counts), _at(kinds), n, max_norm, norm.data_ptr(), ws.data_ptr(), ws.numel())
    return norm


def adam_step_clipped(p, g, m, v, t, max_norm, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-7, norm=None):
    """adam_step over one tensor or lists of float32 tensors with the gradients scaled by min(1, max_norm / global norm) on
    the way (Keras Adam(global_clipnorm=max_norm)); g is left as it is -> the norm before clipping, (1,) float32 on the device.
    max_norm may be infinite (no clipping).  A norm that is not finite makes the step NaN, as an unclipped one would be."""
    max_norm = _max_norm(max_norm)
    if int(t) < 1:
        raise ValueError(f't is the 1-based step count, got {t}')
    dev, n, (pp, gg, mm, vv), counts, kinds = _tensor_lists(p=p, g=g, m=m, v=v)
    if kinds is not None:
        raise TypeError('p, g, m, v: expected torch.float32')
    ws, norm = _norm_buffers(dev, n, norm)
    _call_on(dev, 'ty1_adam_step_clip_f32', _at(pp), _at(gg), _at(mm), _at(vv), _at(counts), n, max_norm, float(lr), float(beta1), float(beta2), float(eps),
             int(t), norm.data_ptr(), ws.data_ptr(), ws.numel())
    return norm


class KernelTimer:
    """HIP-event timing of every library launch on its own stream (bench.py roofline leg)."""

    def __init__(self, only=None, every=1):
        """only: time just the launches whose name starts with this prefix (two event records per launch cost a few
        per cent of a step when every launch is bracketed); every: of those, only every n-th one."""
        self.only, self.every = only, int(every)

    def __enter__(self):
        _lib.call('ty1_prof_reset')
        _lib.call('ty1_prof_filter', self.only.encode() if self.only else b'')
        _lib.call('ty1_prof_stride', self.every)
        _lib.call('ty1_prof_enable', 1)
        return self

    def __exit__(self, *exc):
        _lib.call('ty1_prof_enable', 0)
        _lib.call('ty1_prof_filter', b'')
        _lib.call('ty1_prof_stride', 1)

    @staticmethod
    def table():
        import ctypes
        buf = ctypes.create_string_buffer(16384)
        _lib.call('ty1_prof_dump', buf, len(buf))
        rows = {}
        for line in buf.value.decode().splitlines():
            name, n, ms, flops, nbytes = line.split()
            rows[name] = dict(launches=int(n), ms=float(ms), flops=float(flops), bytes=float(nbytes))
        return rows
