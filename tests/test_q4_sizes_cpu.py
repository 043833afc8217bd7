"""Sizes of caches that no call takes, or that 64 bits do not hold."""
import pytest

MOST = 2**31 - 1


@pytest.mark.parametrize("blocks,layers,n_kv", [(MOST, MOST, MOST), (MOST, MOST, 1), (MOST, 1, 65537), (2**27, 16, 1), (2**20, 36, 65536), (2**30, 1, 2), (MOST, 2**21, 2**12)])
def test_a_cache_of_2_to_the_31_pages_or_more_has_no_size(pkg, blocks, layers, n_kv):
    for group in (32, 64, 128):
        assert pkg.kv4_cache_bytes(blocks, layers, n_kv, 128, group) == 0


def test_the_largest_caches_have_a_size(pkg):
    assert pkg.kv4_cache_bytes(MOST, 1, 1, 128, 32) == MOST * 2304
    assert pkg.kv4_cache_bytes(1, 32767, 65536, 128, 128) == 32767 * 65536 * 2112
    assert pkg.kv4_cache_bytes(2**20, 36, 8, 128, 64) == 2**20 * 36 * 8 * 2176
