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


def test_more_elements_than_one_launch_has_threads_for():
    """A launch holds fewer than 2^32 threads: rows beyond are refused with their reason, not by a launch that fails."""
    lib = nat.load()
    many = 2 ** 31 - 1
    assert lib.clt_mx_quantise(P, many, 96, 96, 1, 0, P, P, None) == RANGE                  # 16 elements a thread
    assert lib.clt_mx_dequantise(P, P, many, 96, 0, P, 96, 1, None) == RANGE                # 8 of two rows
    assert lib.clt_mx_dequantise(P, P, many, 96, 0, P, 96, 0, None) == RANGE                # 4 of two rows in float32
    assert lib.clt_mx_cache_write(P, P, 0, 96, 1, None, 0, 0, many, 96, 1, 1, P, P, many, None, None) == RANGE
    assert lib.clt_mx_cache_read(P, P, many, 1, None, 0, 0, many, 96, 1, 0, None, None, None, None, 1.0, P, P, 0, many, 1, None) == RANGE
    T, d, F = 16 * 65535, 131072, 256
    ws = lib.clt_mx_encode_workspace_bytes(T, d, F, 1, 0)
    assert lib.clt_mx_encode(P, None, P, P, None, P, T, d, F, 1, T * d, 0, T * F, F, 1, P, ws, None) == RANGE
