"""CPU: sizes of the attention decoder's calls whose products pass 64 or 32
bits are refused, or answered with what the true product gives."""
import pytest

from test_decode_cpu import P, refused


@pytest.mark.parametrize("row_stride,outer_stride", [(1 << 60, 64), (1 << 60, (1 << 60) + 64), ((1 << 62) // 3, 1 << 40)])
def test_beam_reorder_refuses_overlap_beyond_64_bits(row_stride, outer_stride):
    """B * K * row_stride passes 2^63: the blocks overlap all the same."""
    import pkc
    why = refused(pkc.beam_reorder, P, P, 65535, 32, row_bytes=64, row_stride=row_stride, n_outer=2, outer_stride=outer_stride)
    assert "overlap" in why
