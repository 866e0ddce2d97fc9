"""How the training operators cut a call (csrc/linear_plan.h), on the host alone."""
import pytest

import linear_plan as plan

SPAN = 0x7fffffff                       # bytes that the 32-bit offsets of a tile reach
BYTES = {'fp32': 4, 'bf16': 2, 'fp16': 2}


def check_pitch(cut, elem, pitch_a, pitch_b):
    """Operands that come by LDS-DMA have rows that the offsets of a 256-row tile reach; the 256 x 256 tile has no other way."""
    assert not cut['a_dma'] or 256 * pitch_a * elem <= SPAN + 256, cut
    assert not cut['b_dma'] or 256 * pitch_b * elem <= SPAN + 256, cut
    assert cut['tile'] < 256 or (cut['a_dma'] and cut['b_dma']), cut


@pytest.mark.parametrize('dtype', BYTES)
@pytest.mark.parametrize('m,n', [(256, 256), (512, 512), (9, 4096), (4096, 520), (1000, 5)])
def test_rows_longer_than_a_tile_reaches(m, n, dtype):
    elem = BYTES[dtype]
    border = SPAN // 256 // elem // 8 * 8
    for k in (border - 8, border, border + 7, border + 8, 4300000, 4300001, 9000000, 16700000):
        pitch = -(-k // 8) * 8
        check_pitch(plan.forward(dtype, m, n, k)['product'], elem, pitch, pitch)
        p = plan.backward(dtype, m, n, k, packed=True, act='gelu', x_act='silu')                 # gx: w [n][k], gw: h [m][k]
        check_pitch(p['gx'], elem, n, pitch)
        check_pitch(p['gw'], elem, n, pitch)
        assert not p['scaled'] or pitch * 2 * 256 <= SPAN
        for act in ('none', 'leaky_relu', 'gelu'):
            p = plan.backward(dtype, m, k, n, act=act)                                           # dz [m][k]
            check_pitch(p['gx'], elem, pitch, n)
            check_pitch(p['gw'], elem, pitch, n)


def test_short_rows_still_come_by_dma():
    """The bound takes nothing from rows under it: copies are made and the largest tile is taken as before."""
    assert plan.forward('bf16', 16384, 4096, 4096)['product'] == {'tile': 256, 'tiles': 1024, 'whole': 1024, 'splits': 1, 'a_dma': 1, 'b_dma': 1}
    assert plan.forward('bf16', 8200, 520, 513)['copies'] == 2
    p = plan.backward('bf16', 16384, 4096, 4096, act='gelu', x_act='gelu', packed=True)
    assert p['scaled'] and p['gx']['tile'] == p['gw']['tile'] == 256
    assert plan.forward('bf16', 512, 512, 4100000)['product']['a_dma']


@pytest.mark.parametrize('elem', [2, 4])
@pytest.mark.parametrize('dma', [True, False])
def test_a_launch_holds_its_blocks(elem, dma):
    """A launch has less than 2^32 lanes along x, 2^24 blocks of 256; products with more tiles take larger ones or none."""
    largest = 0
    for rows in range(20, 44):
        for i in (-1, 0, 77):
            for cols, depth in ((1, 1), (5, 8), (64, 64), (130, 4096), (4096, 4096)):
                cut = plan.product(elem, (1 << rows) + i, cols, depth, dma, dma)
                blocks = cut['whole'] + (cut['tiles'] - cut['whole']) * cut['splits']
                assert blocks * 256 < 1 << 32, cut
                b = cut['tile']
                assert cut['tiles'] in (0, -(-((1 << rows) + i) // b) * -(-cols // b)), cut
                largest = max(largest, blocks)
    assert largest > 1 << 23
