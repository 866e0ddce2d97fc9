"""The training operators at sizes that only their larger tiles and longer paths see, against plain 64-bit formulas on the same card."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import linear_plan as plan  # noqa: E402
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
