"""Requests of the packed operations whose launch would pass the size of a grid are refused, by the query
and by the launch: host code only, no GPU."""
import ctypes as C

from iom_amd import iomx
from test_packed_refusals import INVALID, OVERFLOW, attention_views, launch, query


def test_attention_of_more_workgroups_than_a_grid_has():
    """A launch has fewer than 2^32 lanes: 2^24 - 1 workgroups of 256."""
    rows = 1 << 16
    most = attention_views(Hq=8, Hkv=8, T=rows, D=64, S=4095)                # 512 blocks of 128 rows each
    assert 4095 * 8 * 512 < 1 << 24
    assert query(most, max_rows=rows) == (0, 0, 1)
    past = attention_views(Hq=8, Hkv=8, T=rows, D=64, S=4096)
    assert query(past, max_rows=rows)[0] == OVERFLOW and launch(past, max_rows=rows) == OVERFLOW
    assert query(past, max_rows=rows - 128)[0] == 0                          # a tighter bound on the rows


def test_attention_of_more_tokens_than_are_counted():
    """A row's tokens are counted in 32 bits, 64 at a time (a kernel whose count wraps would not end)."""
    at = dict(Hq=1, Hkv=1, D=8, S=1, N=1, P=16, M=0x7FFFFFF, W=1)
    past = attention_views(T=0x7FFFFFF0, **at)
    assert query(past, max_rows=1)[0] == OVERFLOW and launch(past, max_rows=1) == OVERFLOW
    assert query(attention_views(T=0x7FFFFF00, **at), max_rows=1) == (0, 0, 1)
