"""Microscaled formats: numbers at the C entry points that no buffer can go with are refused before anything is launched."""
from crosslayer_coding_amd import _native as nat

P = 4096                                                # an address nothing is launched on
ARG, RANGE = -1, -6
TOP = 2 ** 63 - 1


def test_rows_whose_end_is_past_what_64_bits_count():
    lib = nat.load()
    for first in (TOP, TOP - 2, 2 ** 62, 9):
        assert lib.clt_mx_cache_write(P, P, 256, 64, 0, None, 0, first, 4, 64, 1, 0, P, P, 8, None, None) == ARG, first
        assert lib.clt_mx_cache_read(P, P, 8, 0, None, 0, first, 4, 64, 1, 0, None, None, None, None, 1.0, P, P, 0, 4, 0, None) == ARG, first
    for out_row in (TOP, TOP - 2, 2 ** 62, 1):
        assert lib.clt_mx_cache_read(P, P, 8, 0, None, 0, 0, 4, 64, 1, 0, None, None, None, None, 1.0, P, P, out_row, 4, 0, None) == ARG, out_row
    assert lib.clt_mx_cache_read(P, P, 8, 0, None, 0, 0, 4, 64, 1, 0, None, None, None, None, 1.0, P, P, 0, 2 ** 60, 0, None) == RANGE
