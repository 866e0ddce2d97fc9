"""The training operators at sizes that only their larger tiles and longer paths see, against plain 64-bit formulas on the same card."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import linear_plan as plan  # noqa: E402
import test_gpu_linear as small_sizes  # noqa: E402
import pifuhd_amd  # noqa: E402,F401
from pifuhd_amd import linear as L  # noqa: E402

DEV = 'cuda'


def whole_numbers(rows, cols, columns, seed, dtype=torch.bfloat16):
    """A matrix of zeros with whole numbers from -2 to 2 in `columns`: sums of its products are exact in 32 bits."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    m = torch.zeros(rows, cols, dtype=dtype, device=DEV)
    m[:, columns] = torch.randint(-2, 3, (rows, len(columns)), generator=g, device=DEV).to(dtype)
    return m


def small(rows, cols, seed, dtype=torch.bfloat16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randint(-3, 4, (rows, cols), generator=g, device=DEV, dtype=torch.int8).to(dtype)


def some_columns(cols):
    return torch.unique(torch.cat([torch.arange(40), torch.arange(0, cols, cols // 60), torch.arange(cols - 40, cols)])).to(DEV)


def test_forward_of_rows_over_8_mib():
    """Rows longer than the 32-bit offsets of a tall tile reach: every row of every tile is its own."""
    m, n, k = 512, 512, 4300000
    assert plan.forward('bf16', m, n, k)['product']['tile'] < 256
    at = some_columns(k)
    x, w = whole_numbers(m, k, at, 1), small(n, k, 2)
    want = x[:, at].double() @ w[:, at].double().t()
    assert torch.equal(L.linear(x, w), want.bfloat16())
    assert torch.equal(L.linear(x[:5], w[:40]), want[:5, :40].bfloat16())


def test_backward_of_rows_over_8_mib():
    m, n, k = 256, 4300000, 256
    assert plan.backward('bf16', m, n, k, act='relu', need=('x',))['gx']['tile'] < 256
    at = some_columns(n)
    g, w, z = whole_numbers(m, n, at, 3), small(n, k, 4), small(m, n, 5)
    gx, _, gb = L.linear_backward(g, None, w, z, act='relu', need=('x', 'bias'))
    dz = g[:, at].double() * (z[:, at] > 0)
    assert torch.equal(gx, (dz @ w[at].double()).bfloat16())
    assert torch.equal(gb[at], dz.sum(0).bfloat16()) and int((gb != 0).sum()) <= len(at)


def test_weight_gradient_of_rows_over_8_mib():
    m, n, k = 40, 24, 4300001
    g, x = small(m, n, 6), small(m, k, 7)
    gw = L.linear_backward(g, x, small(n, k, 8), need=('weight',))[1]
    assert torch.equal(gw, (g.t().float() @ x.float()).bfloat16())           # whole numbers: exact in 32 bits


def test_more_rows_than_a_launch_has_small_tiles():
    """2^30 rows are 2^24 tiles of 64 rows, one launch's worth of lanes and more: larger tiles take them."""
    m, n = (1 << 30) + 77, 5
    assert plan.forward('bf16', m, n, 1)['product']['tile'] > 64
    x = torch.empty(m, 1, dtype=torch.bfloat16, device=DEV)
    step = 1 << 26
    for i in range(0, m, step):
        rows = torch.arange(i, min(i + step, m), device=DEV)
        x[i:i + step, 0] = (rows % 251 - 125).bfloat16()
    w = torch.tensor([[1.0], [-1.0], [2.0], [0.0], [0.5]], device=DEV).bfloat16()
    y = L.linear(x, w)
    gx = L.linear_backward(y, None, w, need=('x',))[0]
    for i in range(0, m, step):
        part = x[i:i + step]
        assert torch.equal(y[i:i + step], part * w.t())
        assert torch.equal(gx[i:i + step], (part.float() * 6.25).bfloat16())


# ---- the tiles that larger products take.  Each case names the cut it is for (tile, whole or split along the sum with or without whole
# tiles before it, which operands come by LDS-DMA), so that another planner cannot leave a kernel untested without a test saying so.
def cut(plan_of_product):
    p = plan_of_product
    kind = 'whole' if p['splits'] == 1 else 'both' if p['whole'] else 'split'
    return f"{p['tile']} {kind} {p['a_dma']}{p['b_dma']}"


def matrix(rows, cols, ld, seed, dtype, numbers):
    """N(0, 1) or whole numbers from -3 to 3, in rows of pitch ld whose other elements are NaN."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    buf = torch.full((rows, ld), float('nan'), dtype=dtype, device=DEV)
    v = buf[:, :cols]
    v.copy_(torch.randint(-3, 4, (rows, cols), generator=g, device=DEV, dtype=torch.int8) if numbers else
            torch.randn(rows, cols, generator=g, device=DEV))
    return v


def close(got, want, tol, what):
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), f'{what}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}'


def own_rounding(got, want, t, what):
    """The error's norm is that of rounding the result to T, and hardly more: operands that keep 11 bits or more add 2 % to bf16's."""
    least = (want.to(t).double() - want).norm()
    assert (got.double() - want).norm() <= 1.1 * least, f'{what}: {float((got.double() - want).norm() / least):.2f} times the rounding of T'


FORWARD = [
    # dtype, m, n, k, extra elements of a row of x and of w, cut
    ('fp32', 3000, 2056, 40, 0, 0, '128 whole 11'), ('fp32', 5000, 777, 41, 0, 0, '128 whole 00'),
    ('fp32', 1030, 777, 4100, 0, 0, '128 split 11'), ('fp32', 4100, 2056, 264, 0, 0, '128 both 11'),
    ('fp32', 2050, 777, 1300, 1, 0, '64 whole 01'), ('fp32', 8200, 1030, 252, 1, 0, '64 both 01'),
    ('bf16', 4100, 1030, 40, 0, 0, '128 whole 11'), ('bf16', 5000, 777, 41, 0, 0, '128 whole 00'),
    ('bf16', 8200, 510, 504, 3, 0, '128 whole 01'), ('fp16', 8200, 510, 504, 0, 3, '128 whole 10'),
    ('fp16', 1300, 777, 4104, 0, 0, '128 split 11'), ('bf16', 4100, 2056, 2000, 0, 0, '128 both 11'),
    ('bf16', 4100, 2056, 1032, 0, 0, '256 whole 11'), ('fp16', 4100, 2056, 1032, 0, 0, '256 whole 11'),
    ('bf16', 2050, 2056, 4104, 0, 0, '256 split 11'), ('fp16', 8200, 2600, 2000, 0, 0, '256 both 11'),
]


@pytest.mark.parametrize('dtype,m,n,k,px,pw,kind', FORWARD, ids=[' '.join(map(str, c[:4])) + ' ' + c[6] for c in FORWARD])
def test_forward_tiles(dtype, m, n, k, px, pw, kind):
    """Whole numbers: exact before the one rounding, so equal bit for bit, with bias and residual, every element its own.  Then N(0, 1)
    with gelu, residual and both kept forms, within the bounds of the small sizes' test."""
    assert cut(plan.forward(dtype, m, n, k, k + px, k + pw)['product']) == kind
    t = small_sizes.TYPES[dtype]
    x, w, r = matrix(m, k, k + px, 1, t, True), matrix(n, k, k + pw, 2, t, True), matrix(m, n, n + 3, 3, t, True)
    b = matrix(1, n, n, 4, t, True)[0]
    z = x.double() @ w.double().t() + b.double()
    y, kept = L.linear(x, w, b, r, act='relu', keep='dense')
    assert torch.equal(kept, z.to(t)) and torch.equal(y, (z.clamp(min=0) + r.double()).to(t))
    assert torch.equal(L.linear(x, w), (z - b.double()).to(t))
    x, w, r = matrix(m, k, k + px, 5, t, False), matrix(n, k, k + pw, 6, t, False) / k ** 0.5, matrix(m, n, n, 7, t, False)
    if pw:
        w = torch.nn.functional.pad(w, (0, pw))[:, :k]
    b = matrix(1, n, n, 8, t, False)[0]
    want, ty, z, tz = small_sizes.forward64(x, w, b, r, 'gelu', t)
    y, kept = L.linear(x, w, b, r, act='gelu', keep='pack8')
    close(y, want, ty, 'y')
    unit = torch.pow(2.0, kept.scales.double() - 127).repeat_interleave(32, 1)[:, :n]
    close(L.unpack8(kept), z, tz * (1 + 2.0 ** -4) + 2.0 ** -4 * z.abs() + 2.0 ** -10 * unit, 'z8')
    again, kept = L.linear(x, w, b, r, act='gelu', keep='dense')
    close(kept, z, tz + small_sizes.rounding(z.abs() + tz, t), 'z')
    assert torch.equal(again, y)


BACKWARD = [
    # dtype, m, n, k, act, x_act, packed, extra elements of a row of grad, cuts of gx and gw, both from scaled fp16
    ('fp32', 2000, 3000, 2056, 'none', 'none', False, 0, '64 both 11', '64 both 11', 0),
    ('fp32', 4100, 520, 2056, 'leaky_relu', 'none', False, 0, '128 both 11', '128 split 11', 0),
    ('fp32', 520, 2056, 4100, 'none', 'none', False, 0, '64 both 11', '128 both 11', 0),
    ('fp32', 4100, 1030, 777, 'relu', 'none', True, 0, '64 both 11', '128 split 11', 0),
    ('fp32', 41, 5000, 777, 'none', 'none', False, 0, '64 split 10', '128 whole 10', 0),
    ('fp32', 40, 3000, 2056, 'relu', 'none', False, 0, '64 split 11', '128 whole 11', 0),
    ('bf16', 4100, 1300, 777, 'none', 'none', False, 1, '64 whole 01', '128 split 01', 0),
    ('bf16', 4100, 130, 1030, 'none', 'none', False, 0, '128 whole 00', '64 split 00', 0),
    ('fp16', 1030, 2050, 2050, 'none', 'none', False, 0, '64 whole 01', '128 whole 01', 0),
    ('bf16', 20000, 1024, 257, 'leaky_relu', 'none', True, 0, '128 whole 11', '128 split 11', 0),
    ('fp16', 2050, 4104, 2056, 'relu', 'none', False, 0, '256 split 11', '128 both 11', 0),
    ('fp16', 4104, 2050, 2056, 'relu', 'none', True, 0, '128 both 11', '256 split 11', 0),
    ('bf16', 2050, 4104, 2056, 'gelu', 'gelu', True, 0, '256 split 11', '128 both 11', 1),
    ('bf16', 4104, 2050, 2056, 'gelu', 'silu', True, 0, '128 both 11', '256 split 11', 1),
    ('bf16', 1032, 4100, 2056, 'gelu', 'tanh', False, 0, '128 split 11', '256 whole 11', 1),
    ('bf16', 8200, 1300, 1030, 'tanh', 'gelu', True, 0, '256 whole 11', '128 split 11', 1),
    ('bf16', 520, 4100, 2056, 'silu', 'silu', False, 0, '128 split 11', '128 whole 11', 1),
    ('bf16', 20000, 264, 1030, 'sigmoid', 'gelu', True, 0, '128 whole 11', '64 split 11', 1),
    ('bf16', 2000, 8200, 2600, 'gelu', 'gelu', True, 0, '256 split 11', '256 both 11', 1),
]


@pytest.mark.parametrize('dtype,m,n,k,act,x_act,packed,pg,kind_x,kind_w,scaled', BACKWARD,
                         ids=[' '.join(map(str, c[:4])) + f' {c[8]} {c[9]}' for c in BACKWARD])
def test_backward_tiles(dtype, m, n, k, act, x_act, packed, pg, kind_x, kind_w, scaled):
    """As the forward test: whole numbers through relu or no activation are exact in checkpoints and sums; two recomputed operands are
    held to the bounds of the small sizes' tests."""
    p = plan.backward(dtype, m, n, k, act, x_act, packed, ldg=n + pg)
    assert (cut(p['gx']), cut(p['gw']), p['scaled']) == (kind_x, kind_w, scaled)
    t = small_sizes.TYPES[dtype]
    if not scaled:
        g, x, w, z = matrix(m, n, n + pg, 1, t, True), matrix(m, k, k, 2, t, True), matrix(n, k, k, 3, t, True), matrix(m, n, n, 4, t, True)
        exact = 'relu' if act == 'leaky_relu' else act
        got = L.linear_backward(g, L.pack8(x) if packed else x, w, (L.pack8(z) if packed else z) if act != 'none' else None, act=exact)
        dz = g.double() if act == 'none' else g.double() * (z > 0)
        for v, want, name in zip(got, (dz @ w.double(), dz.t() @ x.double(), dz.sum(0)), ('gx', 'gw', 'gb')):
            assert torch.equal(v, want.to(t)), name
    g, x, z = matrix(m, n, n + pg, 5, t, False), matrix(m, k, k, 6, t, False), matrix(m, n, n, 8, t, False)
    w = matrix(n, k, k, 7, t, False) / k ** 0.5
    px, pz = (L.pack8(x), L.pack8(z)) if packed else (x, z)
    xv, zv = (L.unpack8(px), L.unpack8(pz)) if packed else (x, z)
    call = lambda: L.linear_backward(g, px, w, pz if act != 'none' else None, act=act, x_act=x_act)      # noqa: E731
    got = call()
    for v, (want, tol), name in zip(got, small_sizes.backward64(g, xv, w, zv, act, False, x_act, t), ('gx', 'gw', 'gb')):
        close(v, want, tol, name)
    if scaled:
        dz, h = g.double() * small_sizes.slope64(zv.double(), act, False), small_sizes.act64(xv.double(), x_act)
        # as in the small sizes' test of two recomputed operands: half an fp16 step of each, and what fp16 cannot hold of the smallest
        e_dz = g.double().abs() * small_sizes.V + 2.0 ** -11 * dz.abs() + 2.0 ** -34 * dz.abs().amax(0)
        e_h = (1 + xv.double().abs()) * small_sizes.V + 2.0 ** -11 * h.abs() + 2.0 ** -34 * h.abs().amax(0)
        want = dz.t() @ h
        tol = (m + 2) * small_sizes.U * ((dz.abs() + e_dz).t() @ (h.abs() + e_h)) + e_dz.t() @ (h.abs() + e_h) + dz.abs().t() @ e_h
        close(got[1], want, tol + small_sizes.rounding(want.abs() + tol, t), 'gw as from fp16')
        own_rounding(got[1], want, t, 'gw')
    assert all(torch.equal(a, c) for a, c in zip(call(), got))


HALVES = [
    # dtype, m, n, k, act, x_act, packed, cuts of gx and gw: dz (a smooth act) and a recomputed x (a smooth x_act) in halves
    ('fp16', 4100, 1030, 1000, 'silu', 'silu', False, '128 both 11', '128 split 11'),
    ('bf16', 8200, 500, 1000, 'tanh', 'sigmoid', False, '128 both 11', '128 split 11'),
    ('bf16', 5000, 520, 1024, 'gelu', 'none', False, '128 whole 11', '64 split 11'),
    ('bf16', 5000, 1024, 520, 'none', 'gelu', True, '64 whole 11', '64 split 11'),
    ('bf16', 5000, 1024, 513, 'leaky_relu', 'silu', True, '64 whole 11', '64 split 11'),
    ('fp16', 300, 2500, 777, 'gelu', 'gelu', False, '64 split 10', '64 whole 11'),
    ('bf16', 4100, 130, 1030, 'sigmoid', 'none', False, '128 whole 10', '64 split 10'),
    ('bf16', 500, 4100, 2000, 'silu', 'silu', False, '128 split 11', '128 both 11'),
    ('fp16', 30000, 128, 257, 'tanh', 'silu', True, '128 whole 10', '64 split 11'),
    ('fp16', 300, 5000, 777, 'gelu', 'gelu', False, '64 split 11', '128 whole 11'),
    ('bf16', 130, 70, 50, 'gelu', 'gelu', True, '64 whole 10', '64 whole 11'),
    ('fp16', 9, 300, 257, 'gelu', 'tanh', False, '64 split 10', '64 whole 11'),
    ('bf16', 1, 1000, 1000, 'silu', 'gelu', True, None, None),
    ('fp16', 2, 5, 3, 'sigmoid', 'gelu', False, None, None),
]


@pytest.mark.parametrize('dtype,m,n,k,act,x_act,packed,kind_x,kind_w', HALVES, ids=[' '.join(map(str, c[:6])) for c in HALVES])
def test_operands_in_halves(dtype, m, n, k, act, x_act, packed, kind_x, kind_w):
    """16-bit operands that were computed on the way in, as two halves each: the gradients are as from fp32 operands, their only 16-bit
    rounding that of the result.  A second half is off by half a step of a value of half a step (bf16: 2^-16 of the whole; fp16: 2^-22,
    or 2^-25), and the product of two second halves, as small, is left out."""
    p = plan.backward(dtype, m, n, k, act, x_act, packed)
    smooth = ('sigmoid', 'tanh', 'gelu', 'silu')
    assert p['halves'] == (act in smooth) + 2 * (x_act in smooth) and not p['scaled']
    assert kind_x is None or (cut(p['gx']), cut(p['gw'])) == (kind_x, kind_w)
    t = small_sizes.TYPES[dtype]
    g, x, z = matrix(m, n, n + 1, 5, t, False), matrix(m, k, k + 3, 6, t, False), matrix(m, n, n + 2, 8, t, False)
    w = matrix(n, k, k, 7, t, False) / k ** 0.5
    px, pz = (L.pack8(x), L.pack8(z)) if packed else (x, z)
    xv, zv = (L.unpack8(px), L.unpack8(pz)) if packed else (x, z)
    call = lambda need: L.linear_backward(g, px, w, pz if act != 'none' else None, act=act, x_act=x_act, need=need)      # noqa: E731
    got = call(('x', 'weight', 'bias'))
    gd, wd = g.double(), w.double()
    dz = gd * small_sizes.slope64(zv.double(), act, False) if act != 'none' else gd
    h = small_sizes.act64(xv.double(), x_act)
    half, least = (2.0 ** -16, 0.0) if t == torch.bfloat16 else (2.0 ** -22, 2.0 ** -25)
    once = small_sizes.rounding(dz, t) if act == 'leaky_relu' else 0.0       # (not in halves: a hundredth of a value is rounded)
    e_dz = (small_sizes.V * gd.abs() + half * dz.abs() + least if act in smooth else small_sizes.U * gd.abs()) + once
    e_h = small_sizes.V * (1 + xv.double().abs()) + half * h.abs() + least if x_act in smooth else torch.zeros_like(h)
    gx, gw, gb = dz @ wd, dz.t() @ h, dz.sum(0)
    lost = half * dz.abs().t() @ h.abs() if act in smooth and x_act in smooth else 0.0
    tx = 2 * (n + 2) * small_sizes.U * ((dz.abs() + e_dz) @ wd.abs()) + e_dz @ wd.abs()
    tw = 3 * (m + 2) * small_sizes.U * ((dz.abs() + e_dz).t() @ (h.abs() + e_h)) + e_dz.t() @ (h.abs() + e_h) + dz.abs().t() @ e_h + lost
    tb = (m + 2) * small_sizes.U * gd.abs().sum(0) + small_sizes.V * gd.abs().sum(0)
    for v, want, tol, name in zip(got, (gx, gw, gb), (tx, tw, tb), ('gx', 'gw', 'gb')):
        close(v, want, tol + small_sizes.rounding(want.abs() + tol, t), name)
        if want.numel() > 1000:
            own_rounding(v, want, t, name)
    assert all(torch.equal(call((name,))[i], got[i]) for i, name in enumerate(('x', 'weight', 'bias')))


@pytest.mark.parametrize('dtype', ['bf16', 'fp16'])
def test_halves_of_large_and_infinite_values(dtype):
    """A dz over the type's largest value is held by its two halves: gradients are finite where their formula is.  Infinities and NaN
    stay in their own row of gx and their own column of dz, not finite."""
    t = small_sizes.TYPES[dtype]
    m, n, k = 40, 24, 32
    most = 60000.0 if t == torch.float16 else 1.7e38
    g, z = torch.ones(m, n, dtype=t, device=DEV), torch.full((m, n), 1.4, device=DEV).to(t)        # gelu'(1.4) = 1.129
    g[3] = most
    x = torch.full((m, k), 2.0 ** -9, device=DEV).to(t)
    w = torch.eye(n, k, device=DEV).to(t) * 2.0 ** -4
    assert plan.backward(dtype, m, n, k, 'gelu')['halves'] == 1
    gx, gw, _ = L.linear_backward(g, x, w, z, act='gelu')
    dz = g.double() * small_sizes.slope64(z.double(), 'gelu', False)
    for v, want in ((gx, dz @ w.double()), (gw, dz.t() @ x.double())):
        close(v, want, 2.0 ** -15 * want.abs() + small_sizes.rounding(want, t), 'finite')
    bad = g.clone()
    bad[7, 5], bad[9, 6] = float('inf'), float('nan')
    hx, hw, hb = L.linear_backward(bad, x, w, z, act='gelu')
    rows, cols = [i for i in range(m) if i not in (7, 9)], [i for i in range(n) if i not in (5, 6)]
    assert torch.equal(hx[rows], gx[rows]) and torch.equal(hw[cols], gw[cols])
    assert not torch.isfinite(hw[[5, 6]]).any() and not torch.isfinite(hb[[5, 6]]).any()
    assert not torch.isfinite(hx[7, 5]) and not torch.isfinite(hx[9, 6])


@pytest.mark.parametrize('act,x_act', [('sigmoid', 'gelu'), ('gelu', 'silu')])
def test_scaled_weight_gradient(act, x_act):
    """A product over the size for halves: columns scaled to fp16.  Columns 2^80 apart, one of zeros, some on their activation's flat
    side, infinities and NaN in their own rows only; the bounds are those of the small sizes' tests of the same."""
    t = torch.bfloat16
    m, n, k = 20000, 264, 1030
    assert plan.backward('bf16', m, n, k, act, x_act)['scaled']
    g, x, z = matrix(m, n, n, 1, t, False), matrix(m, k, k, 2, t, False), matrix(m, n, n, 3, t, False)
    g.copy_(g.double() * torch.pow(2.0, torch.arange(n, device=DEV).double() % 81 - 40))
    g[:, 7] = 0
    flat_z, flat_x = torch.zeros(n, dtype=torch.bool, device=DEV), torch.zeros(k, dtype=torch.bool, device=DEV)
    for c, v in ((5, 9.0), (17, -9.0), (200, -10.0)):
        z[:, c] = (v + 0.25 * z[:, c].float()).to(t)
        flat_z[c] = True
    for c, v in ((3, -8.0), (700, -9.0), (1029, -9.5)):
        x[:, c] = (v + 0.25 * x[:, c].float()).to(t)
        flat_x[c] = True
    g[13, 9], z[13, 9], x[13, ~flat_x] = 3.3e38, 0.0, 2.0 ** -10        # beside the end of the type's range
    w = torch.zeros(n, k, dtype=t, device=DEV)
    call = lambda grad: L.linear_backward(grad, x, w, z, act=act, x_act=x_act, need=('weight', 'bias'))      # noqa: E731
    gw, gb = call(g)[1:]
    gd, xd = g.double(), x.double()
    dz, h = gd * small_sizes.slope64(z.double(), act, False), small_sizes.act64(xd, x_act)
    e_dz = torch.where(flat_z, 2.0 ** -16 * dz.abs(), small_sizes.V * gd.abs()) + 2.0 ** -11 * dz.abs() + 2.0 ** -34 * dz.abs().amax(0)
    e_h = torch.where(flat_x, 2.0 ** -16 * h.abs(), small_sizes.V * (1 + xd.abs())) + 2.0 ** -11 * h.abs() + 2.0 ** -34 * h.abs().amax(0)
    want = dz.t() @ h
    tol = (m + 2) * small_sizes.U * ((dz.abs() + e_dz).t() @ (h.abs() + e_h)) + e_dz.t() @ (h.abs() + e_h) + dz.abs().t() @ e_h
    close(gw, want, tol + small_sizes.rounding(want.abs() + tol, t) + 2.0 ** -133, 'gw')
    assert not gw[7].any() and gw[flat_z].any(1).all() and gw[:, flat_x].any(0).all()
    bad = g.clone()
    bad[11, 3], bad[12, 6] = float('inf'), float('nan')
    hw, hb = call(bad)[1:]
    rest = [i for i in range(n) if i not in (3, 6)]
    assert not torch.isfinite(hw[[3, 6]]).any() and not torch.isfinite(hb[[3, 6]]).any()
    assert torch.equal(hw[rest], gw[rest]) and torch.equal(hb[rest], gb[rest])


@pytest.mark.parametrize('act', ['tanh', 'sigmoid'])
def test_graph_of_a_scaled_backward_pass(act):
    """The derivative from an output, from checkpoints, over the size for halves: gw at its own rounding; captured and replayed with other
    gradients - eager calls between the replays - equal to the eager calls every time."""
    t = torch.bfloat16
    m, n, k = 20000, 264, 1030
    assert plan.backward('bf16', m, n, k, act, 'gelu', True)['scaled']
    x, w = matrix(m, k, k, 2, t, False), matrix(n, k, k, 3, t, False)
    px = L.pack8(x)
    kept = L.pack8(small_sizes.act64(matrix(m, n, n, 4, t, False).double(), act).to(t))
    gs = [matrix(m, n, n, 10 + i, t, False) * 4.0 ** i for i in range(3)]
    run = lambda grad: L.linear_backward(grad, px, w, kept, act=act, from_output=True, x_act='gelu')      # noqa: E731
    want = [run(g) for g in gs]
    for g, got in zip(gs, want):
        dz = g.double() * small_sizes.slope64(L.unpack8(kept).double(), act, True)
        h = small_sizes.act64(L.unpack8(px).double(), 'gelu')
        own_rounding(got[1], dz.t() @ h, t, 'gw')
        own_rounding(got[2], dz.sum(0), t, 'gb')
    static = gs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(static)
    for g, ref in zip(gs + gs[:1], want + want[:1]):
        static.copy_(g)
        graph.replay()
        again = run(g)
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, ref)) and all(torch.equal(a, c) for a, c in zip(again, ref))
