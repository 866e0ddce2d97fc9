"""Loss of the supervised forward (`PIFuMRNet.get_error`, reference `PIFuMRNet.py:253-274`): the weighted, class-balanced
binary cross entropy the reference's training script installs as `criteria['occ']` (`net_util.py:45-66`).

The value alone is a call of the object; `with_grad` gives the value and its gradient (there is no autograd on the HIP path).  The
reductions run in `pifu_bce_loss` / `pifu_bce_loss_grad` (csrc/loss.hip): one pass over the predictions with fixed-order double
accumulation, so the value is reproducible run to run.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib


class CustomBCELoss:
    """Callable with the reference's signature `(pred, gt, gamma, w=None)`.

    pred / gt: device tensors of one shape whose first axis is the batch (`[B, 1, N]` in `get_error`); gamma: `[B]`
    per-sample positive-class weight, ignored when the loss object was built with its own `gamma`; w: `None`, `[B]`
    per-sample weights, or a tensor of pred's shape.  `brock=True` rescales the labels to [-1, 2] (3 gt - 1)."""

    def __init__(self, brock=False, gamma=None):
        self.brock = bool(brock)
        self.gamma = gamma

    def _arguments(self, pred, gt, gamma, w, dtype):
        """What both calls hand to the library: the tensors (the caller keeps them alive until its call has been issued), batch
        size, elements per batch entry, the fixed gamma and whether w has a weight per element."""
        if not pred.is_cuda:
            raise _lib.PifuError(_lib.ERR_INVALID, 'the HIP path needs device tensors (no CPU fallback)')
        dev = pred.device
        p = _as(pred, dtype, dev).contiguous()
        t = _as(gt, torch.float32, dev)
        if t.shape != p.shape:
            t = t.expand_as(p)
        t = t.contiguous()
        batch = p.shape[0]
        n = p.numel() // batch
        g, fixed = None, 0.0
        if self.gamma is None:
            g = _as(gamma, torch.float32, dev).reshape(-1).contiguous()
            if g.numel() != batch:
                raise ValueError(f'gamma must hold one value per batch entry ({batch}), got {g.numel()}')
        else:
            fixed = float(self.gamma)
        wt, per_element = None, 0
        if w is not None:
            wt = _as(w, torch.float32, dev)
            if wt.dim() == 1:
                if wt.numel() != batch:
                    raise ValueError(f'w must hold one value per batch entry ({batch}), got {wt.numel()}')
                wt = wt.contiguous()
            else:
                wt, per_element = wt.expand_as(p).contiguous(), 1
        return p, t, batch, n, g, fixed, wt, per_element

    def __call__(self, pred, gt, gamma, w=None):
        from .nets import _ptr, _stream_ptr
        p, t, batch, n, g, fixed, wt, per_element = self._arguments(pred, gt, gamma, w, torch.float32)
        dev = p.device
        ctx = _ctx_cache(dev)
        out = torch.empty(1, device=dev, dtype=torch.float32)
        _lib.call('pifu_bce_loss', ctx.h, _ptr(p), _ptr(t), batch, n, _ptr(g), C.c_float(fixed), _ptr(wt), per_element,
                  int(self.brock), _ptr(out), _stream_ptr(dev))
        return out[0]

    def with_grad(self, pred, gt, gamma, w=None, scale=1.0):
        """`(scale * loss, scale * d loss / d pred)`: the value a call of the object gives and its gradient, in one pass over the
        tensors.  The gradient has pred's shape and type (float32, bfloat16 or float16; the arithmetic is float32) and is zero
        where the clamp of the predictions to [1e-5, 1 - 1e-5] holds - which includes the zeros that points outside the bounding
        box predict.  A NaN among the predictions makes the value NaN; its own gradient is zero.  `scale`: a factor of the whole
        loss (loss scaling, the mean over several stacks)."""
        if pred.dtype not in DTYPES:
            raise ValueError(f'{pred.dtype} is not supported (float32, bfloat16, float16)')
        if pred.numel() == 0:
            raise _lib.PifuError(_lib.ERR_INVALID, 'empty input (the mean would be nan)')
        p, t, batch, n, g, fixed, wt, per_element = self._arguments(pred, gt, gamma, w, pred.dtype)
        dev = p.device
        out = t.new_empty(())
        grad = torch.empty_like(p)
        ws = t.new_empty(_lib.BCE_WORKSPACE, dtype=torch.uint8)
        _lib.check(_lib.load().pifu_bce_loss_grad(
            _context(dev), DTYPES[p.dtype], p.data_ptr(), t.data_ptr(), batch, n, g.data_ptr() if g is not None else None, fixed,
            wt.data_ptr() if wt is not None else None, per_element, self.brock, float(scale), out.data_ptr(), grad.data_ptr(),
            ws.data_ptr(), _lib.BCE_WORKSPACE, _stream(dev.index)))
        return out, grad

    forward = __call__


def _as(t, dtype, dev):
    return t.detach() if t.dtype == dtype and t.device == dev else t.detach().to(dev, dtype)


DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}

# the raw handle of a device's current stream (torch.cuda.current_stream builds an object around it: 2 us of a 10 us call)
_stream = torch._C._cuda_getCurrentRawStream

_CTXS = {}


def _context(device):
    """The handle of `_ctx_cache(device)` for a tensor's device."""
    ctx = _CTXS.get(device.index)
    return ctx.h if ctx is not None else _ctx_cache(device).h


def _ctx_cache(device):
    """One library context per device for the stand-alone ops of this module.  The first call on a device creates it, which allocates
    memory: not while a graph is being captured, and with the caller's current device put back afterwards."""
    from .nets import _Ctx
    key = torch.device(device).index or 0
    if key not in _CTXS:
        with torch.cuda.device(key):
            if torch.cuda.is_current_stream_capturing():
                raise _lib.PifuError(_lib.ERR_INVALID, f'the first call on device {key} allocates memory: make one before the capture')
            _CTXS[key] = _Ctx(torch.device('cuda', key))
    return _CTXS[key]
