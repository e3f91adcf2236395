"""Shapes of a 4-bit paged cache's pools."""
import pytest

from qweninferenceengine_b200 import ops


def test_whole_blocks():
    assert ops.PagedKVQ4.pool_shape(7, 2, 64, 128) == (7, 2, 4, 2560)
    assert ops.PagedKVQ4.pool_shape(7, 2, 16, 64) == (7, 2, 1, 1280)


@pytest.mark.parametrize("page_size", [0, 8, 24, 72, -16])
def test_pages_that_blocks_do_not_fill(page_size):
    """Pages of 24 slots were given those of 16, and their tables other slots than meant."""
    with pytest.raises(ValueError, match="page_size"):
        ops.PagedKVQ4.pool_shape(7, 2, page_size, 128)
