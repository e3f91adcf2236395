"""Numbers that do not fit the library's 32-bit arguments are refused, not cut (runs
without a GPU: the numbers are looked at before the tensors)."""
import pytest

from qweninferenceengine_b200 import ops

WIDE = 1 << 32   # its low 32 bits are 0


@pytest.mark.parametrize("numbers", [dict(n_select=WIDE + 4), dict(n_select=4, n_first=WIDE),
                                     dict(n_select=4, n_last=WIDE + 1), dict(n_select=WIDE, n_first=WIDE, n_last=0)])
def test_selection(numbers):
    with pytest.raises(ValueError, match="n_select"):
        ops.select_pages(None, None, None, **numbers)


class Pages:
    """prefix_pages of 2^29 numbers, never read."""

    shape, is_contiguous, data_ptr, get_device = (1 << 29,), lambda self: True, lambda self: 0, lambda self: 0
    numel = lambda self: 1 << 29   # noqa: E731


def test_prefix():
    import torch

    class Handle:
        index, page_size, device = 0, 16, "cuda:0"

    pages = Pages()
    pages.dtype = torch.int32
    with pytest.raises(ValueError, match="prefix_len"):
        ops.attention_prefix_paged(Handle(), None, None, pages, WIDE + 16)


def test_listed_pages():
    import torch

    class Handle:
        index, n_seq, n_kv_heads, device = 0, 1, 1, "cuda:0"

    class Lists(Pages):
        dtype, shape = torch.int32, (1, 1, WIDE + 4)

        def dim(self):
            return 3

    with pytest.raises(ValueError, match="pages"):
        ops.attention_sparse_paged(Handle(), None, None, Lists())
