"""Refusals of the training operators that need no GPU: the C entries' argument checks and the Python layer's."""
import ctypes as C

import pytest
import torch

import pifuhd_amd  # noqa: F401
from pifuhd_amd import _lib, linear as L
from pifuhd_amd.net_util import CustomBCELoss

PTR = 1 << 20                      # an address that is never followed: every call below is refused before it would be


def _ctx():
    return C.c_void_p(PTR)


def _forward(**change):
    a = L._LinearArgs()
    a.dtype, a.act, a.m, a.n, a.k = _lib.F32, 0, 4, 8, 16
    a.x, a.ldx, a.w, a.ldw, a.y, a.ldy = PTR, 16, PTR, 16, PTR, 8
    for name, v in change.items():
        setattr(a, name, v)
    return a


def _backward(**change):
    a = L._LinearGradArgs()
    a.dtype, a.act, a.m, a.n, a.k = _lib.BF16, 1, 4, 8, 16
    a.grad, a.ldg, a.x, a.ldx, a.w, a.ldw, a.z, a.ldz = PTR, 8, PTR, 16, PTR, 16, PTR, 8
    a.gx, a.ldgx, a.gw, a.ldgw, a.gb = PTR, 16, PTR, 16, PTR
    for name, v in change.items():
        setattr(a, name, v)
    return a


@pytest.mark.parametrize('change', [
    dict(dtype=3), dict(dtype=-1), dict(act=7), dict(act=-1), dict(m=-1), dict(n=0), dict(k=0), dict(x=None), dict(w=None), dict(y=None),
    dict(ldx=15), dict(ldw=15), dict(ldy=7), dict(x=PTR + 2), dict(bias=PTR + 1), dict(residual=PTR, ldr=7), dict(z=PTR, ldz=7),
    dict(z8=L._Packed8Arg(PTR, 8, None, 1)), dict(z8=L._Packed8Arg(PTR, 7, PTR, 1)), dict(z8=L._Packed8Arg(PTR, 8, PTR, 0)),
    dict(n=1 << 24, ldy=1 << 24), dict(k=1 << 24, ldx=1 << 24, ldw=1 << 24),
])
def test_linear_entry_refuses(change):
    a = _forward(**change)
    lib = _lib.load()
    assert lib.pifu_linear(_ctx(), C.byref(a), None, 0, None) == _lib.ERR_INVALID
    assert b'pifu_linear' in lib.pifu_last_error()
    assert lib.pifu_linear_workspace(_ctx(), C.byref(a)) == _lib.ERR_INVALID
    assert lib.pifu_linear(None, C.byref(_forward()), None, 0, None) == _lib.ERR_INVALID
    assert lib.pifu_linear(_ctx(), None, None, 0, None) == _lib.ERR_INVALID


@pytest.mark.parametrize('change', [
    dict(dtype=3), dict(act=7), dict(x_act=9), dict(act=5, from_output=1), dict(act=6, from_output=1), dict(m=-1), dict(n=0), dict(k=0),
    dict(grad=None), dict(z=None), dict(x=None), dict(w=None), dict(ldg=7), dict(ldx=15), dict(ldw=15), dict(ldz=7), dict(ldgx=15),
    dict(ldgw=15), dict(grad=PTR + 1), dict(gb=PTR + 1), dict(z=None, z8=L._Packed8Arg(PTR, 8, None, 1)),
    dict(x=None, x8=L._Packed8Arg(PTR, 15, PTR, 1)), dict(n=1 << 24, ldg=1 << 24, ldz=1 << 24),
])
def test_linear_backward_entry_refuses(change):
    a = _backward(**change)
    lib = _lib.load()
    assert lib.pifu_linear_backward(_ctx(), C.byref(a), C.c_void_p(PTR), 1 << 40, None) == _lib.ERR_INVALID
    assert b'pifu_linear_backward' in lib.pifu_last_error()
    assert lib.pifu_linear_backward_workspace(_ctx(), C.byref(a)) == _lib.ERR_INVALID


def test_linear_backward_entry_refuses_a_small_workspace():
    lib = _lib.load()
    a = _backward()
    need = lib.pifu_linear_backward_workspace(_ctx(), C.byref(a))
    assert need > 0
    assert lib.pifu_linear_backward(_ctx(), C.byref(a), C.c_void_p(PTR), need - 1, None) == _lib.ERR_NOMEM
    assert lib.pifu_linear_backward(_ctx(), C.byref(a), None, need, None) == _lib.ERR_NOMEM
    assert lib.pifu_linear_backward(_ctx(), C.byref(a), C.c_void_p(PTR + 8), need, None) == _lib.ERR_INVALID


def test_workspace_of_a_few_rows_is_none():
    lib = _lib.load()
    for m in (1, _lib.LINEAR_FEW_ROWS):
        assert lib.pifu_linear_workspace(_ctx(), C.byref(_forward(m=m, k=4096, ldx=4096, ldw=4096))) == 0
    assert lib.pifu_linear_workspace(_ctx(), C.byref(_forward(m=_lib.LINEAR_FEW_ROWS + 1, k=4096, ldx=4096, ldw=4096))) > 0


def test_empty_batch_is_no_launch():
    lib = _lib.load()
    assert lib.pifu_linear(_ctx(), C.byref(_forward(m=0, x=None, y=None)), None, 0, None) == _lib.OK
    p = L._Packed8Arg(None, 8, None, 1)
    assert lib.pifu_pack8(_ctx(), _lib.F32, None, 8, 0, 8, C.byref(p), None) == _lib.OK


@pytest.mark.parametrize('dtype,ldx,rows,cols,packed,x', [
    (3, 8, 4, 8, (PTR, 8, PTR, 1), PTR), (0, 7, 4, 8, (PTR, 8, PTR, 1), PTR), (0, 8, -1, 8, (PTR, 8, PTR, 1), PTR),
    (0, 8, 4, 0, (PTR, 8, PTR, 1), PTR), (0, 8, 4, 8, (None, 8, PTR, 1), PTR), (0, 8, 4, 8, (PTR, 8, None, 1), PTR),
    (0, 8, 4, 8, (PTR, 7, PTR, 1), PTR), (0, 33, 4, 33, (PTR, 33, PTR, 1), PTR), (0, 8, 4, 8, (PTR, 8, PTR, 1), None),
    (1, 8, 4, 8, (PTR, 8, PTR, 1), PTR + 1),
])
def test_pack8_entries_refuse(dtype, ldx, rows, cols, packed, x):
    lib = _lib.load()
    p = L._Packed8Arg(*packed)
    assert lib.pifu_pack8(_ctx(), dtype, x, ldx, rows, cols, C.byref(p), None) == _lib.ERR_INVALID
    assert lib.pifu_unpack8(_ctx(), dtype, C.byref(p), rows, cols, x, ldx, None) == _lib.ERR_INVALID
    assert lib.pifu_pack8(_ctx(), dtype, x, ldx, rows, cols, None, None) == _lib.ERR_INVALID


def test_bce_loss_grad_entry_refuses():
    lib = _lib.load()

    def call(ctx=PTR, dtype=0, pred=PTR, gt=PTR, batch=1, n=8, out=PTR, grad=PTR, ws=PTR, ws_bytes=_lib.BCE_WORKSPACE):
        return lib.pifu_bce_loss_grad(ctx, dtype, pred, gt, batch, n, None, 0.5, None, 0, 0, 1.0, out, grad, ws, ws_bytes, None)
    for bad in (dict(ctx=None), dict(dtype=5), dict(pred=None), dict(gt=None), dict(batch=0), dict(n=0), dict(grad=None), dict(ws=PTR + 4)):
        assert call(**bad) == _lib.ERR_INVALID, bad
    assert call(ws=None) == _lib.ERR_NOMEM
    assert call(ws_bytes=_lib.BCE_WORKSPACE - 1) == _lib.ERR_NOMEM


def test_host_tensors_are_refused():
    x, w = torch.zeros(4, 16), torch.zeros(8, 16)
    for call in (lambda: L.linear(x, w), lambda: L.linear_backward(torch.zeros(4, 8), x, w), lambda: L.pack8(x),
                 lambda: L.unpack8(L.Packed8(torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8))),
                 lambda: CustomBCELoss().with_grad(torch.zeros(1, 1, 4), torch.zeros(1, 1, 4), torch.tensor([0.5]))):
        with pytest.raises(_lib.PifuError, match='device tensors'):
            call()


def test_checkpoint_shapes():
    codes, scales = torch.zeros(4, 70, dtype=torch.uint8), torch.zeros(4, 3, dtype=torch.uint8)
    p = L.Packed8(codes, scales)
    assert p.nbytes == 4 * 73 and tuple(p.shape) == (4, 70)
    v = p.columns(32, 70)
    assert tuple(v.codes.shape) == (4, 38) and tuple(v.scales.shape) == (4, 2) and v.codes.data_ptr() == codes.data_ptr() + 32
    assert tuple(p.columns(0, 33).scales.shape) == (4, 2)
    for first, last in ((1, 64), (32, 32), (0, 71), (-32, 32)):
        with pytest.raises(ValueError):
            p.columns(first, last)
    for c, s in ((codes, scales[:, :2]), (codes, scales[:3]), (codes.float(), scales), (codes[0], scales)):
        with pytest.raises(ValueError):
            L.Packed8(c, s)


def test_overlap_of_matrices():
    """Whether two views of one buffer share an element, against the elements themselves."""
    buf = torch.zeros(400, dtype=torch.bfloat16)

    def elements(offset, rows, cols, ld):
        return {offset + i * ld + j for i in range(rows) for j in range(cols)}
    shapes = [(o, r, c, ld) for o in (0, 1, 5, 7, 12, 26) for r in (1, 2, 3) for c in (1, 4, 8) for ld in (8, 12, 13) if ld >= c]
    shared = refused = 0
    for a in shapes:
        for b in shapes:
            va, vb = (buf.as_strided((r, c), (ld, 1), o) for o, r, c, ld in (a, b))
            got = L._overlap(va, a[3] if a[1] > 1 else a[2], vb, b[3] if b[1] > 1 else b[2])
            want = bool(elements(*a) & elements(*b))
            if a[3] != b[3] and a[1] > 1 and b[1] > 1:
                assert got or not want, (a, b)               # different pitches: never missed, sometimes refused
                refused += got and not want
            else:
                assert got == want, (a, b)
            shared += want
    assert shared > 1000 and refused > 0


def test_first_call_on_a_device(monkeypatch):
    """A device's context is created under that device, the caller's is current again afterwards, and no capture is broken by it."""
    from pifuhd_amd import net_util, nets
    current, made = [0], []

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *_):
            current[0] = self.before

    class Ctx:
        def __init__(self, device):
            assert device.index == current[0]
            made.append(device.index)
    monkeypatch.setattr(net_util, '_CTXS', {})
    monkeypatch.setattr(nets, '_Ctx', Ctx)
    monkeypatch.setattr(torch.cuda, 'device', Device)
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: True)
    with pytest.raises(_lib.PifuError, match='before the capture'):
        net_util._ctx_cache(torch.device('cuda', 3))
    assert not made and current == [0]
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: False)
    first = net_util._ctx_cache(torch.device('cuda', 3))
    assert made == [3] and current == [0] and net_util._ctx_cache(torch.device('cuda', 3)) is first


def test_products_of_more_than_a_launch_are_refused():
    """By the workspace query and by the call, before anything is launched."""
    lib = _lib.load()
    for a, query, entry in ((_forward(m=1 << 40), lib.pifu_linear_workspace, lib.pifu_linear),
                            (_backward(m=1 << 40), lib.pifu_linear_backward_workspace, lib.pifu_linear_backward),
                            (_backward(m=1 << 40, gw=None, gb=None), lib.pifu_linear_backward_workspace, lib.pifu_linear_backward)):
        assert query(_ctx(), C.byref(a)) == _lib.ERR_INVALID
        assert b'more outputs than one launch' in lib.pifu_last_error()
        assert entry(_ctx(), C.byref(a), C.c_void_p(PTR), 1 << 60, None) == _lib.ERR_INVALID
    assert lib.pifu_linear_workspace(_ctx(), C.byref(_forward(m=1 << 30))) >= 0


def test_unpack8_of_rows_longer_than_a_launch_is_refused():
    """2^24 - 1 blocks of 512 columns are the most; the longest rows under that fit."""
    lib = _lib.load()
    most = ((1 << 24) - 1) * 512
    for cols in (most + 1, 1 << 34, 1 << 38):
        p = L._Packed8Arg(PTR, cols, PTR, -(-cols // 32))
        for rows in (1, 5):
            assert lib.pifu_unpack8(_ctx(), _lib.BF16, C.byref(p), rows, cols, PTR, cols, None) == _lib.ERR_INVALID
            assert b'one launch' in lib.pifu_last_error()
