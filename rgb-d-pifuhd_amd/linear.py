"""Training operators of the surface classifier: the layers of `MLP.forward` (`MLP.py:43-75`) as operators of their own, their
gradients, and 8-bit checkpoints of activations between the two passes.

    y, z = linear(x, weight, bias, act='leaky_relu', keep='pack8')         # z: a Packed8, a quarter of fp32's bytes
    gx, gw, gb = linear_backward(grad, pack8(x), weight, z, act='leaky_relu')

As everywhere in this package there is no autograd: gradients are explicit calls.  A tensor that requires grad is refused here while
grad mode is on instead of being cut out of the graph silently.  Device tensors only (no CPU fallback); every tensor of a call has
one type (float32, bfloat16 or float16) and lives on one device, whose current torch stream the kernels run on.  All calls but a
device's first one may be captured into a graph: their only scratch memory is a torch tensor of the call's own.  (A captured graph
whose memory pool is shared with another one must not replay at the same time as that one: torch's own rule.)
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from .net_util import DTYPES, _context, _stream

ACTS = {'none': 0, 'relu': 1, 'leaky_relu': 2, 'sigmoid': 3, 'tanh': 4, 'gelu': 5, 'silu': 6}
FROM_OUTPUT = ('none', 'relu', 'leaky_relu', 'sigmoid', 'tanh')       # activations whose derivative follows from their output
PACK8_BLOCK = 32                          # PIFU_PACK8_BLOCK


class Packed8:
    """An 8-bit checkpoint of a matrix [rows, cols]: `codes` uint8 [rows, cols] (e4m3) and `scales` uint8 [rows, ceil(cols / 32)],
    one power of two per 32 consecutive columns of a row (`pifu_packed8` in include/pifuhd_hip.h).  Both may be strided views with
    unit column stride; `columns()` gives such a view.  A view that ends inside a block shares its last scale with the columns behind
    it: it is for reading, not for packing into."""
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
        p = cls.__new__(cls)                                 # (nothing to check)
        p.codes = torch.empty((rows, cols), dtype=torch.uint8, device=device)
        p.scales = torch.empty((rows, -(-cols // PACK8_BLOCK)), dtype=torch.uint8, device=device)
        return p

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
    """t [..., C] as [rows, C] with unit column stride - a view where the strides allow it, a copy otherwise - and its row pitch."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    rows, cols = t.shape
    ld, step = t.stride()
    if rows < 2:
        ld = cols
    if (step != 1 and cols > 1) or ld < cols:
        return t.contiguous(), cols                          # (a broadcast gradient - stride 0 - is written out)
    return t, ld


def _ld(t, what, rows, cols, device):
    """The row pitch of a matrix that is used where it lies."""
    if t.shape != (rows, cols) or t.device != device:
        raise ValueError(f'{what} is {tuple(t.shape)} on {t.device}, expected {(rows, cols)} on {device}')
    ld, step = t.stride()
    if rows < 2:
        ld = cols
    if (step != 1 and cols > 1) or ld < cols:
        raise ValueError(f'{what}, strides {t.stride()}: unit column stride and rows that do not overlap are needed')
    return ld


def _span(t, ld):
    first = t.data_ptr()
    return first, first + ((t.shape[0] - 1) * ld + t.shape[1]) * t.element_size() if t.numel() else first


def _overlap(a, lda, b, ldb):
    """Whether two matrices of one element type share an element.  Rows of one pitch may interleave (columns of one buffer) without
    sharing any; of two different pitches, spans that cross count as an overlap."""
    (lo, hi), (first, last) = _span(a, lda), _span(b, ldb)
    if first >= hi or lo >= last:
        return False
    if lda != ldb and a.shape[0] > 1 and b.shape[0] > 1:
        return True
    ld = lda if a.shape[0] > 1 else ldb if b.shape[0] > 1 else last - lo + hi - first        # (one row has no pitch of its own)
    at, odd = divmod(first - lo, a.element_size())
    if odd:
        return True
    rows, col = divmod(at, ld)                               # b's first element in the grid of a's rows
    return (col < a.shape[1] and -b.shape[0] < rows < a.shape[0]) or \
           (ld - col < b.shape[1] and -b.shape[0] < rows + 1 < a.shape[0])


def _packed(p, rows, cols, what, device):
    return _Packed8Arg(p.codes.data_ptr(), _ld(p.codes, what, rows, cols, device),
                       p.scales.data_ptr(), _ld(p.scales, f'{what} (scales)', rows, -(-cols // PACK8_BLOCK), device))


def _fresh(p, cols):
    """`_packed` of a checkpoint just made."""
    return _Packed8Arg(p.codes.data_ptr(), cols, p.scales.data_ptr(), -(-cols // PACK8_BLOCK))


def _run(workspace, entry, args, like, device):
    """Calls `entry` with a workspace of the size that `workspace` (None: none is needed) names."""
    ctx, args = _context(device), C.byref(args)
    need = workspace(ctx, args) if workspace is not None else 0
    if need < 0:
        _lib.check(need)
    ws = like.new_empty(need, dtype=torch.uint8) if need else None
    _lib.check(entry(ctx, args, ws.data_ptr() if need else None, need, _stream(device.index)))


def pack8(x, out=None):
    """The 8-bit checkpoint of x [..., C] (leading axes flattened) -> `Packed8` (`pifu_pack8`)."""
    device = _device_of(x, 'x')
    code = _dtype_code(x.dtype)
    _same(x, 'x', x.dtype, device)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f'x {tuple(x.shape)}: at least one column')
    t, ld = _rows(x)
    rows, cols = t.shape
    if out is None:
        out = Packed8.empty(rows, cols, device)
        arg = _fresh(out, cols)
    else:
        arg = _packed(out, rows, cols, 'out', device)
    _lib.check(_lib.load().pifu_pack8(_context(device), code, t.data_ptr(), ld, rows, cols, C.byref(arg), _stream(device.index)))
    return out


def unpack8(packed, dtype=torch.float32, out=None):
    """The values a checkpoint stands for, [rows, cols] of `dtype` (exact in float32 and bfloat16; float16 where they are in its
    range) (`pifu_unpack8`)."""
    device = _device_of(packed.codes, 'codes')
    code = _dtype_code(dtype if out is None else out.dtype)
    rows, cols = packed.shape
    if out is None:
        out, ld = torch.empty((rows, cols), dtype=dtype, device=device), cols
    else:
        _same(out, 'out', out.dtype, device)
        ld = _ld(out, 'out', rows, cols, device)
    arg = _packed(packed, rows, cols, 'packed', device)
    _lib.check(_lib.load().pifu_unpack8(_context(device), code, C.byref(arg), rows, cols, out.data_ptr(), ld, _stream(device.index)))
    return out


def linear(x, weight, bias=None, residual=None, act='none', keep=None, out=None):
    """act(x weight^T + bias) + residual (`pifu_linear`): x [..., K], weight [N, K], bias [N], residual [..., N] -> [..., N].

    act: 'none', 'relu', 'leaky_relu' (slope 0.01), 'sigmoid', 'tanh', 'gelu' (erf) or 'silu'.  keep: None; 'dense' or 'pack8' return
    `(y, z)` with the pre-activation z = x weight^T + bias as a tensor [..., N] or as a `Packed8` [rows, N] written by the same
    kernel.  out: a matrix [rows, N] with unit column stride to receive y, e.g. the leading columns of the next layer's wider input,
    whose trailing columns may be x; it may be the residual itself, but must not share elements with x, the weight or the bias."""
    device = _device_of(x, 'x')
    dtype = x.dtype
    code, act = _dtype_code(dtype), _act_code(act)
    _same(x, 'x', dtype, device)
    _same(weight, 'weight', dtype, device)
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1] or weight.numel() == 0:
        raise ValueError(f'x {tuple(x.shape)} and weight {tuple(weight.shape)} do not multiply: x [..., K], weight [N, K]')
    n, k = weight.shape
    (xr, ldx), (w, ldw) = _rows(x), _rows(weight)
    m = xr.shape[0]
    b = r = z = None
    ldr = 0
    if bias is not None:
        _same(bias, 'bias', dtype, device)
        if bias.shape != (n,):
            raise ValueError(f'bias {tuple(bias.shape)}: expected {(n,)}')
        b = bias.contiguous()
    if residual is not None:
        _same(residual, 'residual', dtype, device)
        if residual.shape != (*x.shape[:-1], n):
            raise ValueError(f'residual {tuple(residual.shape)}: expected {(*x.shape[:-1], n)}')
        r, ldr = _rows(residual)
    if out is None:
        y, ldy = x.new_empty((m, n)), n
    else:
        _same(out, 'out', dtype, device)
        y, ldy = out, _ld(out, 'out', m, n, device)
        for what, t, ld in (('x', xr, ldx), ('weight', w, ldw), ('bias', b, n), ('residual', r, ldr)):
            if t is None or (what == 'residual' and t.data_ptr() == y.data_ptr() and (ld == ldy or m < 2)):
                continue
            if _overlap(y, ldy, t if t.dim() == 2 else t[None], ld):
                raise ValueError(f'out overlaps {what}')
    z8 = ()
    if keep == 'dense':
        z = x.new_empty((m, n))
    elif keep == 'pack8':
        kept = Packed8.empty(m, n, device)
        z8 = _fresh(kept, n)
    elif keep is not None:
        raise ValueError(f"keep must be None, 'dense' or 'pack8', got {keep!r}")
    if m:
        lib = _lib.load()
        args = _LinearArgs(code, act, m, n, k, xr.data_ptr(), ldx, w.data_ptr(), ldw, b.data_ptr() if b is not None else None,
                           r.data_ptr() if r is not None else None, ldr, y.data_ptr(), ldy, z.data_ptr() if z is not None else None, n, z8)
        _run(lib.pifu_linear_workspace if m > _lib.LINEAR_FEW_ROWS else None, lib.pifu_linear, args, xr, device)
    if x.dim() != 2:
        if out is None:
            y = y.view(*x.shape[:-1], n)
        if z is not None:
            z = z.view(*x.shape[:-1], n)
    if keep is None:
        return y
    return y, z if keep == 'dense' else kept


def linear_backward(grad, x, weight, kept=None, act='none', from_output=False, x_act='none', need=('x', 'weight', 'bias')):
    """The gradients of `linear` for grad = dL/dy [..., N] -> `(gx [..., K], gw [N, K], gb [N])`, None for those not in `need`
    (`pifu_linear_backward`).  The residual's gradient is `grad` itself.

    x: the layer's input, a tensor [..., K] or a `Packed8` [rows, K] (None if 'weight' is not needed).  kept: the pre-activation the
    forward pass kept, a tensor [..., N] or a `Packed8` [rows, N] (None for act='none'); with from_output=True the activation's
    OUTPUT instead, before any residual was added ('relu', 'leaky_relu', 'sigmoid' and 'tanh' only) - for a chain of layers that is
    the next layer's input, so one checkpoint per layer serves both.  x_act: activation to apply to x first, for an x that is the
    previous layer's kept pre-activation (gx is the gradient behind that activation, i.e. the previous layer's grad).

    bfloat16 and float16, more than 4 outputs: dz = grad * act' of a smooth activation and an input recomputed through one enter the
    products as two 16-bit halves each (rows * N * K up to 2^32, results rounded once) or rounded to 16 bits (larger: results off by up
    to 1.4 times their rounding; the header says which and where gw is scaled instead).  float16 has its own range there: |dz| over
    65504 (in halves 131008) becomes infinite and under 2^-25 zero, so scale the loss as for any float16 step."""
    device = _device_of(grad, 'grad')
    dtype = grad.dtype
    code, act_code, x_act_code = _dtype_code(dtype), _act_code(act), _act_code(x_act)
    if from_output and act not in FROM_OUTPUT:
        raise ValueError(f'the derivative of {act!r} does not follow from its output: keep the pre-activation')
    need = set(need)
    if not need or not need <= {'x', 'weight', 'bias'}:
        raise ValueError(f"need: any of 'x', 'weight', 'bias', got {sorted(need)}")
    _same(grad, 'grad', dtype, device)
    _same(weight, 'weight', dtype, device)
    if weight.dim() != 2 or weight.numel() == 0 or grad.dim() < 1 or grad.shape[-1] != weight.shape[0]:
        raise ValueError(f'grad {tuple(grad.shape)} and weight {tuple(weight.shape)} do not fit: grad [..., N], weight [N, K]')
    n, k = weight.shape
    (g, ldg), (w, ldw) = _rows(grad), _rows(weight)
    m = g.shape[0]
    gx = gw = gb = xr = zr = None
    ldx = ldz = 0
    x8 = z8 = ()
    if 'weight' in need:
        if x is None:
            raise ValueError('the gradient of the weight needs x')
        if isinstance(x, Packed8):
            x8 = _packed(x, m, k, 'x', device)
        else:
            _same(x, 'x', dtype, device)
            if x.shape != (*grad.shape[:-1], k):
                raise ValueError(f'x {tuple(x.shape)}: expected {(*grad.shape[:-1], k)}')
            xr, ldx = _rows(x)
        gw = w.new_empty((n, k))
    if act != 'none':
        if kept is None:
            raise ValueError(f'the derivative of {act!r} needs what the forward pass kept')
        if isinstance(kept, Packed8):
            z8 = _packed(kept, m, n, 'kept', device)
        else:
            _same(kept, 'kept', dtype, device)
            if kept.shape != grad.shape:
                raise ValueError(f'kept {tuple(kept.shape)}: expected {tuple(grad.shape)}')
            zr, ldz = _rows(kept)
    if 'x' in need:
        gx = g.new_empty((m, k))
    if 'bias' in need:
        gb = g.new_empty(n)
    lib = _lib.load()
    args = _LinearGradArgs(code, act_code, bool(from_output), x_act_code, m, n, k, g.data_ptr(), ldg,
                           xr.data_ptr() if xr is not None else None, ldx, x8, w.data_ptr(), ldw,
                           zr.data_ptr() if zr is not None else None, ldz, z8, gx.data_ptr() if gx is not None else None, k,
                           gw.data_ptr() if gw is not None else None, k, gb.data_ptr() if gb is not None else None)
    _run(lib.pifu_linear_backward_workspace, lib.pifu_linear_backward, args, g, device)
    if gx is not None and grad.dim() != 2:
        gx = gx.view(*grad.shape[:-1], k)
    return gx, gw, gb
