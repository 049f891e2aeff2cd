"""Low-rank adapters of the Dense layer: many fine-tuned heads served and trained beside one shared weight.

The Dense layer is the only trainable layer of the network (/root/reference/models/model_tiny_yolov1.py:96; every conv and
BatchNormalization layer is frozen), so a detector fine-tuned for one camera or customer differs from the shared one in 73.8 MB
of weights.  An adapter keeps that difference as W + scale * B^T A of rank R (0.9 MB at rank 16), and one batch may hold images
of any mixture of adapters.  The reference has one set of weights and no counterpart."""
import operator

import numpy as np
import torch

from . import ops


class AdapterBank:
    """`count` adapters of rank `rank` for a DeviceModel's Dense layer: a (count, rank, features) and b (count, rank, units) as
    views of one flat float32 buffer (`flat`, what an optimiser updates in one launch; b's rows are padded to 16 bytes), and
    scale (count).  a starts uniform in +-1/sqrt(features), b at zero: a new adapter changes nothing.  Give a bank and one index
    per image (bank.index(...)) to DeviceModel.predict / detect / head, or train it with engine.AdapterTrainer.  For a bf16
    model the products read a bf16 copy: call changed() after writing to a or b yourself."""

    def __init__(self, model, count, rank, scale=1.0, seed=1):
        count, rank = int(count), int(rank)
        if not (1 <= count <= ops.MAX_ADAPTERS and 1 <= rank <= ops.MAX_RANK):
            raise ValueError(f'{count} adapters of rank {rank}: 1 to {ops.MAX_ADAPTERS} of rank 1 to {ops.MAX_RANK} are supported')
        self.count, self.rank, self.features, self.units, self.device = count, rank, model.K, model.units, model.device
        ldb, n_a = ops.round_up(self.units, 4), count * rank * self.features
        self.flat = torch.zeros(ops.round_up(n_a, 4) + count * rank * ldb, dtype=torch.float32, device=self.device)
        self.a, self.b = self.views(self.flat)
        gen = torch.Generator().manual_seed(seed)
        self.a.copy_((torch.rand((count, rank, self.features), generator=gen) * 2 - 1) * self.features ** -0.5)
        self.scale = torch.full((count,), float(scale), dtype=torch.float32, device=self.device)
        self._bf16 = torch.zeros_like(self.flat, dtype=torch.bfloat16) if getattr(model, 'dtype', 'f32') == 'bf16' else None
        self.changed()

    def views(self, flat):
        """a- and b-shaped views of a flat buffer of this bank's size (its gradients, its moments)."""
        n_a = self.count * self.rank * self.features
        a = flat[:n_a].view(self.count, self.rank, self.features)
        return a, flat[ops.round_up(n_a, 4):ops.round_up(n_a, 4) + self.count * self.rank * ops.round_up(self.units, 4)].view(
            self.count, self.rank, ops.round_up(self.units, 4))[:, :, :self.units]

    def changed(self):
        """a or b were written to: bring the bf16 copy of a bf16 model's bank up to date, in place, and wait for it (any stream may
        read it next, and graphs that were captured with it read the new values)."""
        if self._bf16 is not None:
            with torch.cuda.device(self.device):       # (the cast goes to the current device's stream)
                ops.cast_bf16(self.flat, out=self._bf16)
                torch.cuda.current_stream().synchronize()

    def weights(self, dtype):
        """(a, b) for products in torch.float32 or, in a bf16 model's bank, torch.bfloat16."""
        if dtype == torch.float32:
            return self.a, self.b
        if self._bf16 is None:
            raise ValueError('the bank was made for a float32 model')
        return self.views(self._bf16)

    def index(self, which):
        """Adapter numbers on the host, one per image (-1 or None: the shared weights alone) -> checked int32 tensor on the GPU."""
        which = [-1 if w is None else w for w in (which.tolist() if hasattr(which, 'tolist') else which)]
        for w in which:
            if not isinstance(w, (int, np.integer)) or isinstance(w, bool) or not -1 <= w < self.count:
                raise ValueError(f'adapter {w!r}: expected -1 (none) or 0 to {self.count - 1}')
        return torch.tensor(which, dtype=torch.int32).to(self.device)

    def _check(self, i):
        if isinstance(i, bool):
            raise TypeError(f'adapter {i}: expected a number')
        if not 0 <= operator.index(i) < self.count:
            raise IndexError(f'adapter {i}: the bank has {self.count}')
        return operator.index(i)

    def set(self, i, a, b, scale=None):
        """Store one adapter from host arrays: a (r, features), b (r, units) with r <= rank (the ranks behind r become zero)."""
        i, scale = self._check(i), None if scale is None else float(scale)
        a, b = (torch.as_tensor(np.ascontiguousarray(v, np.float32)) for v in (a, b))
        r = a.shape[0]
        if a.dim() != 2 or r > self.rank or tuple(a.shape) != (r, self.features) or tuple(b.shape) != (r, self.units):
            raise ValueError(f'adapter: a {tuple(a.shape)}, b {tuple(b.shape)} are not (r, {self.features}) and (r, {self.units}) with r <= {self.rank}')
        self.a[i].zero_(); self.b[i].zero_()
        self.a[i, :r].copy_(a); self.b[i, :r].copy_(b)
        if scale is not None:
            self.scale[i] = scale
        self.changed()

    def get(self, i):
        """-> a (rank, features), b (rank, units) as NumPy arrays, scale: what set() takes (and np.savez stores)."""
        i = self._check(i)
        return self.a[i].cpu().numpy(), self.b[i].cpu().numpy(), float(self.scale[i])
