"""What lq_reorder_beams refuses before any launch (made-up addresses, never read)."""
import pytest

from layer_quant_amd import _abi
from test_beam_decode import F32, I64, U8, fake, reorder


@pytest.mark.parametrize("shape,stride", [
    ((8, 16), (8, 1)),             # windows of 16 bytes at every 8
    ((8, 16), (15, 1)),
    ((8, 3, 5), (1, 8, 8)),
    ((8, 4, 6), (6, 3, 1)),        # rows of windows
    ((8, 4, 6), (100, 5, 1)),
    ((8, 2, 3, 4), (200, 10, 4, 2)),
    ((8, 2, 40, 64), (5120, 2560, 63, 1))])
def test_elements_that_overlap(shape, stride):
    b = fake((2, 4), I64)
    assert reorder([fake(shape, U8, stride, data=0x900000)], b) == -1
    assert "overlap" in _abi.last_error()
    assert reorder([fake(shape, F32, stride, data=0x900000)], b) == -1


@pytest.mark.parametrize("shape,stride", [
    ((8, 16), (1, 8)), ((8, 3, 5), (7, 100, 1)), ((8, 1, 6), (6, 0, 1)), ((8, 3, 2, 4), (4, 32, 100, 1)),
    ((8, 2, 4), (9, 4, 1))])
def test_any_order_without_an_overlap(shape, stride):
    """Rows innermost, gaps, extents of one: passed on (one beam per prompt, so nothing is launched)."""
    assert reorder([fake(shape, U8, stride, data=0x900000)], fake((8, 1), I64)) == 0


def test_launch_limits_before_the_first_launch():
    """A tensor that no launch takes is refused before any other is moved, wherever it stands in the list."""
    P = 1 << 20
    b = fake((P, 2), I64)
    small = fake((2 * P, 16), U8, data=0x10000000)
    wide = fake((2 * P, 140000), U8, data=0x1000000000)  # 18 workgroups of 8 KiB for each of 2^20 prompts
    for tensors in ([wide], [small, wide], [wide, small]):
        assert reorder(tensors, b) == -2
        assert "launch limits" in _abi.last_error()
    assert reorder([fake((2 * P, 140000), U8, data=0x1000000000)], fake((2 * P, 1), I64)) == 0  # nothing moves
