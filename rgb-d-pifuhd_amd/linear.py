"""Training operators of the surface classifier: the layers of `MLP.forward` (`MLP.py:43-75`) as operators of their own, their
gradients, and 8-bit checkpoints of activations between the two passes.

    y, z = linear(x, weight, bias, act='leaky_relu', keep='pack8')         # z: a Packed8, a quarter of fp32's bytes
    gx, gw, gb = linear_backward(grad, pack8(x), weight, z, act='leaky_relu')

As everywhere in this package there is no autograd: gradients are explicit calls, and a tensor that requires grad is refused while
grad mode is on instead of being cut out of the graph silently.  Device tensors only (no CPU fallback); every tensor of a call has
one type (float32, bfloat16 or float16) and lives on one device, whose current torch stream the kernels run on.  All calls may be
captured into a graph: their only scratch memory is a torch tensor of the call's own.  (A captured graph whose memory pool is
shared with another one must not replay at the same time as that one: torch's own rule.)
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib

ACTS = {'none': 0, 'relu': 1, 'leaky_relu': 2, 'sigmoid': 3, 'tanh': 4, 'gelu': 5, 'silu': 6}
FROM_OUTPUT = ('none', 'relu', 'leaky_relu', 'sigmoid', 'tanh')       # activations whose derivative follows from their output
DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
PACK8_BLOCK = 32                          # PIFU_PACK8_BLOCK


class Packed8:
    """An 8-bit checkpoint of a matrix [rows, cols]: `codes` uint8 [rows, cols] (e4m3) and `scales` uint8 [rows, ceil(cols / 32)],
    one power of two per 32 consecutive columns of a row (`pifu_packed8` in include/pifuhd_hip.h).  Both may be strided views with
    unit column stride; `columns()` gives such a view."""
    __slots__ = ('codes', 'scales')

    def __init__(self, codes, scales):
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or codes.dim() != 2 or scales.dim() != 2:
            raise ValueError('a checkpoint is two uint8 matrices: codes [rows, cols] and scales [rows, ceil(cols / 32)]')
        if scales.shape[0] != codes.shape[0] or scales.shape[1] != -(-codes.shape[1] // PACK8_BLOCK):
            raise ValueError(f'scales {tuple(scales.shape)} do not fit codes {tuple(codes.shape)}')
        if scales.device != codes.device:
            raise ValueError('codes and scales live on different devices')
        self.codes, self.scales = codes, scales

    @classmethod
    def empty(cls, rows, cols, device):
        return cls(torch.empty(rows, cols, dtype=torch.uint8, device=device),
                   torch.empty(rows, -(-cols // PACK8_BLOCK), dtype=torch.uint8, device=device))

    @property
    def shape(self):
        return self.codes.shape

    @property
    def nbytes(self):
        return self.codes.numel() + self.scales.numel()

    def columns(self, first, last):
        """The checkpoint of columns [first, last), a view; `first` must start a block."""
        if first % PACK8_BLOCK or not 0 <= first < last <= self.codes.shape[1]:
            raise ValueError(f'columns [{first}, {last}) of {tuple(self.codes.shape)}: the first must be a multiple of {PACK8_BLOCK}')
        return Packed8(self.codes[:, first:last], self.scales[:, first // PACK8_BLOCK:-(-last // PACK8_BLOCK)])


class _Packed8Arg(C.Structure):
    _fields_ = [('codes', C.c_void_p), ('ld', C.c_int64), ('scales', C.c_void_p), ('ld_scales', C.c_int64)]


class _LinearArgs(C.Structure):
    _fields_ = [('dtype', C.c_int32), ('act', C.c_int32), ('m', C.c_int64), ('n', C.c_int64), ('k', C.c_int64),
                ('x', C.c_void_p), ('ldx', C.c_int64), ('w', C.c_void_p), ('ldw', C.c_int64), ('bias', C.c_void_p),
                ('residual', C.c_void_p), ('ldr', C.c_int64), ('y', C.c_void_p), ('ldy', C.c_int64),
                ('z', C.c_void_p), ('ldz', C.c_int64), ('z8', _Packed8Arg)]


class _LinearGradArgs(C.Structure):
    _fields_ = [('dtype', C.c_int32), ('act', C.c_int32), ('from_output', C.c_int32), ('x_act', C.c_int32),
                ('m', C.c_int64), ('n', C.c_int64), ('k', C.c_int64), ('grad', C.c_void_p), ('ldg', C.c_int64),
                ('x', C.c_void_p), ('ldx', C.c_int64), ('x8', _Packed8Arg), ('w', C.c_void_p), ('ldw', C.c_int64),
                ('z', C.c_void_p), ('ldz', C.c_int64), ('z8', _Packed8Arg), ('gx', C.c_void_p), ('ldgx', C.c_int64),
                ('gw', C.c_void_p), ('ldgw', C.c_int64), ('gb', C.c_void_p)]


def _device_of(t, what):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f'{what} must be a tensor, got {type(t).__name__}')
    if not t.is_cuda:
        raise _lib.PifuError(_lib.ERR_INVALID, 'the HIP path needs device tensors (no CPU fallback)')
    return t.device


def _same(t, what, dtype, device):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f'{what} must be a tensor, got {type(t).__name__}')
    if t.dtype != dtype or t.device != device:
        raise ValueError(f'{what} is {t.dtype} on {t.device}: every tensor of a call has one type and device ({dtype} on {device})')
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f'{what} requires grad: there is no autograd on the HIP path - call under torch.no_grad() and use the '
                         f'explicit backward calls')


def _dtype_code(dtype):
    code = DTYPES.get(dtype)
    if code is None:
        raise ValueError(f'{dtype} is not supported (float32, bfloat16, float16)')
    return code


def _act_code(act):
    code = ACTS.get(act)
    if code is None:
        raise ValueError(f'unknown activation {act!r} (one of {", ".join(ACTS)})')
    return code


def _rows(t):
    """t [..., C] as [rows, C] with unit column stride: a view where the strides allow it, a copy otherwise."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    if (t.stride(1) != 1 and t.shape[1] > 1) or (t.stride(0) < t.shape[1] and t.shape[0] > 1):
        t = t.contiguous()                                   # (a broadcast gradient - stride 0 - is written out)
    return t


def _ld(t):
    return max(t.stride(0), t.shape[1]) if t.shape[0] > 1 else t.shape[1]


def _span(t):
    first = t.data_ptr()
    return first, first + ((t.shape[0] - 1) * t.stride(0) + t.shape[1]) * t.element_size() if t.numel() else first


def _context(device):
    from .net_util import _ctx_cache
    return _ctx_cache(device).h


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


def _packed(p, rows, cols, what, device):
    if tuple(p.shape) != (rows, cols):
        raise ValueError(f'{what} holds {tuple(p.shape)} values, expected {(rows, cols)}')
    if p.codes.device != device:
        raise ValueError(f'{what} is on {p.codes.device}, the other tensors on {device}')
    codes, scales = p.codes, p.scales
    for t in (codes, scales):
        if (t.stride(1) != 1 and t.shape[1] > 1) or (t.stride(0) < t.shape[1] and t.shape[0] > 1):
            raise ValueError(f'{what}: codes and scales need unit column stride and rows that do not overlap')
    return _Packed8Arg(codes.data_ptr(), _ld(codes), scales.data_ptr(), _ld(scales))


def _workspace(name, ctx, args, device):
    need = getattr(_lib.load(), name)(ctx, C.byref(args))
    if need < 0:
        _lib.check(need)
    return torch.empty(need, dtype=torch.uint8, device=device) if need else None


def pack8(x, out=None):
    """The 8-bit checkpoint of x [..., C] (leading axes flattened) -> `Packed8` (`pifu_pack8`)."""
    device = _device_of(x, 'x')
    code = _dtype_code(x.dtype)
    _same(x, 'x', x.dtype, device)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f'x {tuple(x.shape)}: at least one column')
    t = _rows(x)
    rows, cols = t.shape
    out = Packed8.empty(rows, cols, device) if out is None else out
    arg = _packed(out, rows, cols, 'out', device)
    _lib.call('pifu_pack8', _context(device), code, t.data_ptr(), _ld(t), rows, cols, C.byref(arg), _stream(device))
    return out


def unpack8(packed, dtype=torch.float32, out=None):
    """The values a checkpoint stands for, [rows, cols] of `dtype` (exact in float32 and bfloat16; float16 where they are in its
    range) (`pifu_unpack8`)."""
    device = _device_of(packed.codes, 'codes')
    code = _dtype_code(dtype if out is None else out.dtype)
    rows, cols = packed.shape
    if out is None:
        out = torch.empty(rows, cols, dtype=dtype, device=device)
    elif tuple(out.shape) != (rows, cols) or out.device != device or (out.stride(1) != 1 and cols > 1) or (out.stride(0) < cols and rows > 1):
        raise ValueError(f'out must be [{rows}, {cols}] on {device} with unit column stride')
    arg = _packed(packed, rows, cols, 'packed', device)
    _lib.call('pifu_unpack8', _context(device), code, C.byref(arg), rows, cols, out.data_ptr(), _ld(out), _stream(device))
    return out


def linear(x, weight, bias=None, residual=None, act='none', keep=None, out=None):
    """act(x weight^T + bias) + residual (`pifu_linear`): x [..., K], weight [N, K], bias [N], residual [..., N] -> [..., N].

    act: 'none', 'relu', 'leaky_relu' (slope 0.01), 'sigmoid', 'tanh', 'gelu' (erf) or 'silu'.  keep: None; 'dense' or 'pack8' return
    `(y, z)` with the pre-activation z = x weight^T + bias as a tensor [..., N] or as a `Packed8` [rows, N] written by the same
    kernel.  out: a matrix [rows, N] with unit column stride (e.g. the leading columns of the next layer's wider input) to receive y;
    it may be the residual itself, but must not overlap x or the weight."""
    device = _device_of(x, 'x')
    dtype = x.dtype
    a = _LinearArgs()
    a.dtype, a.act = _dtype_code(dtype), _act_code(act)
    _same(x, 'x', dtype, device)
    _same(weight, 'weight', dtype, device)
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1] or weight.numel() == 0:
        raise ValueError(f'x {tuple(x.shape)} and weight {tuple(weight.shape)} do not multiply: x [..., K], weight [N, K]')
    n, k = weight.shape
    xr, w = _rows(x), _rows(weight)
    m = xr.shape[0]
    shape = (*x.shape[:-1], n)
    a.m, a.n, a.k = m, n, k
    a.x, a.ldx, a.w, a.ldw = xr.data_ptr(), _ld(xr), w.data_ptr(), _ld(w)
    if bias is not None:
        _same(bias, 'bias', dtype, device)
        if tuple(bias.shape) != (n,):
            raise ValueError(f'bias {tuple(bias.shape)}: expected {(n,)}')
        b = bias.contiguous()
        a.bias = b.data_ptr()
    if residual is not None:
        _same(residual, 'residual', dtype, device)
        if tuple(residual.shape) != shape:
            raise ValueError(f'residual {tuple(residual.shape)}: expected {shape}')
        r = _rows(residual)
        a.residual, a.ldr = r.data_ptr(), _ld(r)
    if out is None:
        y = torch.empty(m, n, dtype=dtype, device=device)
    else:
        _same(out, 'out', dtype, device)
        if tuple(out.shape) != (m, n) or (out.stride(1) != 1 and n > 1) or (out.stride(0) < n and m > 1):
            raise ValueError(f'out {tuple(out.shape)}, strides {out.stride()}: expected a matrix {(m, n)} with unit column stride')
        y = out
        lo, hi = _span(y)
        inputs = [('x', xr), ('weight', w)] + ([('bias', b[None])] if bias is not None else [])
        if residual is not None and (r.data_ptr(), _ld(r)) != (y.data_ptr(), _ld(y)):
            inputs.append(('residual', r))
        for what, t in inputs:
            first, last = _span(t)
            if first < hi and lo < last:
                raise ValueError(f'out overlaps {what}')
    a.y, a.ldy = y.data_ptr(), _ld(y)
    z = None
    if keep == 'dense':
        z = torch.empty(m, n, dtype=dtype, device=device)
        a.z, a.ldz = z.data_ptr(), n
    elif keep == 'pack8':
        z = Packed8.empty(m, n, device)
        a.z8 = _packed(z, m, n, 'z', device)
    elif keep is not None:
        raise ValueError(f"keep must be None, 'dense' or 'pack8', got {keep!r}")
    if m:
        ctx = _context(device)
        ws = _workspace('pifu_linear_workspace', ctx, a, device)
        _lib.call('pifu_linear', ctx, C.byref(a), ws.data_ptr() if ws is not None else None, ws.numel() if ws is not None else 0,
                  _stream(device))
    if out is None:
        y = y.view(shape)
    if keep is None:
        return y
    return y, z.view(shape) if keep == 'dense' else z


def linear_backward(grad, x, weight, kept=None, act='none', from_output=False, x_act='none', need=('x', 'weight', 'bias')):
    """The gradients of `linear` for grad = dL/dy [..., N] -> `(gx [..., K], gw [N, K], gb [N])`, None for those not in `need`
    (`pifu_linear_backward`).  The residual's gradient is `grad` itself.

    x: the layer's input, a tensor [..., K] or a `Packed8` [rows, K] (None if 'weight' is not needed).  kept: the pre-activation the
    forward pass kept, a tensor [..., N] or a `Packed8` [rows, N] (None for act='none'); with from_output=True the activation's
    OUTPUT instead, before any residual was added ('relu', 'leaky_relu', 'sigmoid' and 'tanh' only) - for a chain of layers that is
    the next layer's input, so one checkpoint per layer serves both.  x_act: activation to apply to x first, for an x that is the
    previous layer's kept pre-activation (gx is the gradient behind that activation, i.e. the previous layer's grad)."""
    device = _device_of(grad, 'grad')
    dtype = grad.dtype
    a = _LinearGradArgs()
    a.dtype, a.act, a.x_act = _dtype_code(dtype), _act_code(act), _act_code(x_act)
    if from_output and act not in FROM_OUTPUT:
        raise ValueError(f'the derivative of {act!r} does not follow from its output: keep the pre-activation')
    a.from_output = int(bool(from_output))
    need = set(need)
    if not need or not need <= {'x', 'weight', 'bias'}:
        raise ValueError(f"need: any of 'x', 'weight', 'bias', got {sorted(need)}")
    _same(grad, 'grad', dtype, device)
    _same(weight, 'weight', dtype, device)
    if weight.dim() != 2 or weight.numel() == 0 or grad.dim() < 1 or grad.shape[-1] != weight.shape[0]:
        raise ValueError(f'grad {tuple(grad.shape)} and weight {tuple(weight.shape)} do not fit: grad [..., N], weight [N, K]')
    n, k = weight.shape
    g, w = _rows(grad), _rows(weight)
    m = g.shape[0]
    a.m, a.n, a.k = m, n, k
    a.grad, a.ldg, a.w, a.ldw = g.data_ptr(), _ld(g), w.data_ptr(), _ld(w)
    if 'weight' in need:
        if x is None:
            raise ValueError('the gradient of the weight needs x')
        if isinstance(x, Packed8):
            a.x8 = _packed(x, m, k, 'x', device)
        else:
            _same(x, 'x', dtype, device)
            if tuple(x.shape) != (*grad.shape[:-1], k):
                raise ValueError(f'x {tuple(x.shape)}: expected {(*grad.shape[:-1], k)}')
            xr = _rows(x)
            a.x, a.ldx = xr.data_ptr(), _ld(xr)
    if act != 'none':
        if kept is None:
            raise ValueError(f'the derivative of {act!r} needs what the forward pass kept')
        if isinstance(kept, Packed8):
            a.z8 = _packed(kept, m, n, 'kept', device)
        else:
            _same(kept, 'kept', dtype, device)
            if tuple(kept.shape) != tuple(grad.shape):
                raise ValueError(f'kept {tuple(kept.shape)}: expected {tuple(grad.shape)}')
            zr = _rows(kept)
            a.z, a.ldz = zr.data_ptr(), _ld(zr)
    gx = gw = gb = None
    if 'x' in need:
        gx = torch.empty(m, k, dtype=dtype, device=device)
        a.gx, a.ldgx = gx.data_ptr(), k
    if 'weight' in need:
        gw = torch.empty(n, k, dtype=dtype, device=device)
        a.gw, a.ldgw = gw.data_ptr(), k
    if 'bias' in need:
        gb = torch.empty(n, dtype=dtype, device=device)
        a.gb = gb.data_ptr()
    ctx = _context(device)
    ws = _workspace('pifu_linear_backward_workspace', ctx, a, device)
    _lib.call('pifu_linear_backward', ctx, C.byref(a), ws.data_ptr() if ws is not None else None, ws.numel() if ws is not None else 0,
              _stream(device))
    return gx.view(*grad.shape[:-1], k) if gx is not None else None, gw, gb
