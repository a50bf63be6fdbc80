"""Limits of the window attention and KV cache entry points as documented, on the
CPU (tests/launch_log.py): the largest calls launch, the next ones are refused."""
import pytest

from prichs_amd import _lib as L
from tests import launch_log as ll

ITEMS = (1 << 28) - 16  # of one cache call: batch * n * n_kv_heads


def cache_call(name, batch, n, kv):
    """(status, launches) of a cache write or read."""
    return ll.run(f"""
rc = lib.prichs_kv_cache_{name}(P, 4, P, 2, P, None, P, 128 * {kv}, P, 128 * {kv}, {batch}, {n}, {kv},
                                128, 1, None)
result = [rc, launches()]
""")


@pytest.mark.parametrize("name", ["write", "read"])
def test_items_of_a_cache_call(name):
    rc, got = cache_call(name, 1, ITEMS, 1)
    assert rc == L.PRICHS_OK and len(got) == 1
    (_, _, grid, block, _, _), = got
    assert grid[0] * block < 1 << 32 and grid[0] * block // 16 == ITEMS
    for batch, n, kv in ((1, ITEMS + 1, 1), (1, (1 << 28) - 1, 1), (3, ((1 << 28) - 1) // 3, 1),
                         (5, ((1 << 28) - 1) // 15, 3)):
        assert ITEMS < batch * n * kv < 1 << 28
        assert cache_call(name, batch, n, kv) == [L.PRICHS_ERR_INVALID_ARGUMENT, []], (batch, n, kv)
