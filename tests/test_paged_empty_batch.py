"""Calls over a cache without sequences: nothing to do, whatever an empty tensor's address
is (null; runs without a GPU)."""
import test_paged_refusals as refusals
from qweninferenceengine_b200 import _lib


def test_no_sequences_and_only_null_addresses():
    kv = refusals.kv(n_seq=0, page_table=None)
    nothing = dict(q=None, lens=None, ws=None, bytes=0)
    assert refusals.paged(kv, out=None, **nothing) == _lib.QWEN_OK
    assert refusals.prefix(kv, out=None, **nothing) == _lib.QWEN_OK
    assert refusals.select(kv, pages=None, **nothing) == _lib.QWEN_OK
    assert refusals.sparse(kv, pages=None, out=None, **nothing) == _lib.QWEN_OK


def test_what_is_wrong_with_sizes_is_still_refused():
    kv = refusals.kv(n_seq=0, page_table=None)
    refusals.refused(refusals.sparse, kv, "n_select", n=0)
    refusals.refused(refusals.sparse, refusals.kv(n_seq=0, head_dim=96), "head_dim", pages=None)
    refusals.refused(refusals.sparse, refusals.kv(), "null pages", pages=None)
