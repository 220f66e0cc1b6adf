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


@pytest.mark.parametrize("heads,max_q", [(512, (1 << 30) + 1), (1 << 20, (1 << 31) - 1)])
def test_loose_bounds_of_many_heads_count_every_row(heads, max_q):
    """Rows of an item and key head (max_q * heads) whose tiles pass 2^31: the
    number of tiles does not wrap to a few, for which parts of the keys and a
    workspace would be asked."""
    import pkc
    assert pkc.cross_attention_workspace(1, max_q, 20000, heads, 1, 64) == 0
    assert pkc.kv8_attention_workspace(pkc.KV8Cache(k=P, v=P, k_scale=P, v_scale=P, table=P, n_pages=8, page=16, n_kv_heads=1,
                                                    head_dim=64, table_ld=4096), 1, max_q, 20000, heads) == 0
