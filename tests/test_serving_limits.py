"""Sizes at which counts of 32 bits in the serving operators' kernels would end: refused before anything reaches a GPU."""
import ctypes

import pytest

from test_serving_refusals import BASE, NO_DEVICE, cache, decode, made_up_addresses_stay_off_a_gpu  # noqa: F401


def ranges(rows, max_pos, kv_heads, heads):
    """Attention over a cache whose rows are cut into ranges, with a workspace, as far as a call gets."""
    from rptc_b200 import lib
    c = cache(rows=rows, max_pos=max_pos, kv_heads=kv_heads)
    need = lib().rptc_attn_decode_kv4_workspace_bytes(ctypes.byref(c), heads)
    assert need > 0
    return decode(c, heads=heads, ld_q=heads * 128, ld_out=heads * 128, ws=BASE, ws_bytes=need)


def units(rows, max_pos, kv_heads, heads):
    """What all rows' heads are worth when full: tiles of 32 positions and 24 more, for every eight q heads of a kv head."""
    return rows * kv_heads * -(-heads // kv_heads // 8) * (-(-max_pos // 32) + 24)


@pytest.mark.parametrize("rows,max_pos,kv_heads,heads", [(16, 1 << 24, 1, 4096), (65535, 1 << 20, 8, 64), (65535, 4096, 4096, 4096), (16, 16776448 + 1, 1, 4096)])
def test_rows_whose_units_pass_32_bits(rows, max_pos, kv_heads, heads):
    assert units(rows, max_pos, kv_heads, heads) >= 1 << 32
    assert ranges(rows, max_pos, kv_heads, heads) == -7


@pytest.mark.parametrize("rows,max_pos,kv_heads,heads", [(15, 1 << 24, 1, 4096), (64, 1 << 24, 1, 128), (65535, 2049, 8, 64), (16, 16776448 - 32, 1, 4096), (1, 1 << 24, 4096, 4096)])
def test_the_largest_that_are_counted(rows, max_pos, kv_heads, heads):
    assert units(rows, max_pos, kv_heads, heads) < 1 << 32
    assert ranges(rows, max_pos, kv_heads, heads) in NO_DEVICE
