"""The workspace queries answer 0 for every size that the call itself will refuse (runs
without a GPU), and the wrappers do not remember such an answer for other calls."""
import ctypes

import pytest

import test_paged_refusals as refusals
from qweninferenceengine_b200._lib import QWEN_ERR_INVALID_ARGUMENT, lib

SIZES = [dict(dtype=2), dict(dtype=-1), dict(head_dim=96), dict(head_dim=0), dict(page_size=8), dict(page_size=48),
         dict(page_size=512), dict(page_size=0), dict(n_pages=0), dict(n_pages=(1 << 30) + 1), dict(n_seq=65536),
         dict(max_pages=0), dict(max_pages=(1 << 20) + 1, table_stride=1 << 21), dict(table_stride=7),
         dict(n_kv_heads=0), dict(n_kv_heads=1025)]


def queries(kv, heads=12, prefix_len=100, n_select=4):
    s = ctypes.byref(kv)
    return {refusals.paged: lib().qwen_attention_paged_workspace(s, heads),
            refusals.prefix: lib().qwen_attention_prefix_paged_workspace(s, heads, prefix_len),
            refusals.select: lib().qwen_select_pages_workspace(s),
            refusals.sparse: lib().qwen_attention_sparse_paged_workspace(s, heads, n_select)}


@pytest.mark.parametrize("fields", SIZES)
def test_no_workspace_for_sizes_that_are_refused(fields):
    kv = refusals.kv(**fields)
    heads = kv.n_kv_heads or 12
    for call, need in queries(kv, heads).items():
        assert call(kv, heads=heads, qs=1 << 20, os=1 << 20) == QWEN_ERR_INVALID_ARGUMENT
        assert need == 0, call.__name__


@pytest.mark.parametrize("heads", [0, 13, 130])
def test_no_workspace_for_heads_that_are_refused(heads):
    kv = refusals.kv()
    for call, need in queries(kv, heads).items():
        if call is not refusals.select:   # its query is not told the heads
            refusals.refused(call, kv, "n_heads", heads=heads)
            assert need == 0


def test_no_workspace_for_more_tiles_than_a_call_takes():
    kv = refusals.kv(n_seq=65535, n_kv_heads=1024, head_stride=128, max_pages=1 << 16, table_stride=1 << 16)
    rows = dict(heads=1024, qs=131072, os=131072)
    need = queries(kv, 1024, n_select=1 << 20)
    for call, more in ((refusals.paged, {}), (refusals.prefix, {}), (refusals.sparse, dict(n=1 << 20))):
        refusals.refused(call, kv, "more than one call", **rows, **more)
        assert need[call] == 0
    assert queries(kv, 1024, n_select=4)[refusals.sparse] > 0   # a few listed pages of the same cache


def test_no_workspace_for_lengths_that_are_refused():
    kv = refusals.kv()
    assert queries(kv, prefix_len=(1 << 24) + 1)[refusals.prefix] == 0
    refusals.refused(refusals.sparse, kv, "n_select", n=(1 << 20) + 1)
    for n in (0, (1 << 20) + 1):
        assert queries(kv, n_select=n)[refusals.sparse] == 0


def test_addresses_are_not_looked_at():
    bare = refusals.kv(k=None, v=None, bounds=None, page_table=None, page_stride=0, pos_stride=0, head_stride=0)
    assert queries(bare) == queries(refusals.kv()) and 0 not in queries(bare).values()


def test_an_answer_of_zero_is_not_remembered():
    """The same (n_seq, heads, dim, max_pages) with a page size that is refused, then one that is not."""
    from qweninferenceengine_b200 import ops

    class Handle:
        sizes = ("not a device", 3, 2, 128, 8)

        def __init__(self, **fields):
            self.kv = refusals.kv(**fields)
            self.ref = ctypes.byref(self.kv)

    assert ops._workspace_need(Handle(page_size=48), "qwen_attention_paged_workspace", 12) == 0
    need = ops._workspace_need(Handle(), "qwen_attention_paged_workspace", 12)
    assert need == queries(refusals.kv())[refusals.paged]
