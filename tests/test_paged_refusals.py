"""Arguments that the paged-cache entry points refuse before they touch a device
(runs without a GPU): the buffers are made-up addresses that nothing reads."""
import ctypes

import pytest

from qweninferenceengine_b200 import _lib
from qweninferenceengine_b200._lib import QWEN_ERR_INVALID_ARGUMENT, PagedKVStruct, lib

A = 0x10000   # a 256-byte aligned address


def kv(**fields):
    s = PagedKVStruct(A, A, A, A, 16 * 2 * 128, 2 * 128, 128, 64, 16, 2, 128, 3, 8, 8, _lib.QWEN_DTYPE_F16)
    for name, value in fields.items():
        setattr(s, name, value)
    return s


def append(s, **o):
    a = dict(q=A, qs=1536, k=A, ks=256, v=A, vs=256, out=A, os=1536, heads=12, n=3, lens=A, cu=None,
             inv=A, rot=128, inter=0) | o
    return lib().qwen_rope_append_paged(ctypes.byref(s) if s else None, a["q"], a["qs"], a["k"], a["ks"],
                                        a["v"], a["vs"], a["out"], a["os"], a["heads"], a["n"], a["lens"],
                                        a["cu"], a["inv"], a["rot"], a["inter"], None)


def paged(s, **o):
    a = dict(q=A, qs=1536, out=A, os=1536, lse=None, heads=12, lens=A, ws=A, bytes=1 << 40) | o
    return lib().qwen_attention_paged(ctypes.byref(s) if s else None, a["q"], a["qs"], a["out"], a["os"],
                                      a["lse"], a["heads"], a["lens"], 0.1, a["ws"], a["bytes"], None)


def prefix(s, **o):
    a = dict(q=A, qs=1536, out=A, os=1536, lse=None, heads=12, lens=A, pages=A, len=100, ws=A,
             bytes=1 << 40) | o
    return lib().qwen_attention_prefix_paged(ctypes.byref(s) if s else None, a["q"], a["qs"], a["out"],
                                             a["os"], a["lse"], a["heads"], a["lens"], a["pages"], a["len"],
                                             0.1, a["ws"], a["bytes"], None)


def select(s, **o):
    a = dict(q=A, qs=1536, heads=12, lens=A, n=4, first=1, last=1, pages=A, ws=A, bytes=1 << 40) | o
    return lib().qwen_select_pages(ctypes.byref(s) if s else None, a["q"], a["qs"], a["heads"], a["lens"],
                                   a["n"], a["first"], a["last"], a["pages"], a["ws"], a["bytes"], None)


def sparse(s, **o):
    a = dict(pages=A, n=4, q=A, qs=1536, out=A, os=1536, lse=None, heads=12, lens=A, ws=A,
             bytes=1 << 40) | o
    return lib().qwen_attention_sparse_paged(ctypes.byref(s) if s else None, a["pages"], a["n"], a["q"],
                                             a["qs"], a["out"], a["os"], a["lse"], a["heads"], a["lens"],
                                             0.1, a["ws"], a["bytes"], None)


OPS = [append, paged, prefix, select, sparse]


def refused(call, s, text, **o):
    assert call(s, **o) == QWEN_ERR_INVALID_ARGUMENT
    assert text in lib().qwen_last_error().decode()


@pytest.mark.parametrize("call", OPS)
@pytest.mark.parametrize("fields,text", [
    (dict(k=None), "null cache"), (dict(v=None), "null cache"), (dict(page_table=None), "null cache"),
    (dict(dtype=2), "dtype"), (dict(dtype=-1), "dtype"), (dict(head_dim=96), "head_dim"),
    (dict(page_size=8), "page_size"), (dict(page_size=48), "page_size"), (dict(page_size=512), "page_size"),
    (dict(page_size=0), "page_size"), (dict(n_pages=0), "n_pages"), (dict(n_seq=65536), "n_seq"),
    (dict(max_pages=0), "max_pages"), (dict(max_pages=1 << 21, table_stride=1 << 21), "max_pages"),
    (dict(table_stride=7), "table_stride"), (dict(n_kv_heads=5), "n_heads"), (dict(n_kv_heads=0), "n_heads"),
    (dict(page_stride=0), "stride"), (dict(pos_stride=-256), "stride"), (dict(head_stride=132), "stride"),
    (dict(k=A + 8), "aligned"), (dict(v=A + 2), "aligned"), (dict(bounds=A + 8), "aligned")])
def test_cache_descriptions(call, fields, text):
    refused(call, kv(**fields), text)


@pytest.mark.parametrize("call", OPS)
def test_rows_and_lengths(call):
    refused(call, None, "null kv")
    refused(call, kv(), "null q", q=None)
    refused(call, kv(), "q must", q=A + 8)
    refused(call, kv(), "q must", qs=1540)
    refused(call, kv(), "q must", qs=1528)
    refused(call, kv(), "seq_len", lens=None)
    refused(call, kv(), "n_heads", heads=13)
    refused(call, kv(), "n_heads", heads=0)
    refused(call, kv(), "n_heads", heads=130)


@pytest.mark.parametrize("call", [paged, prefix, sparse])
def test_outputs_and_workspace(call):
    refused(call, kv(), "null out", out=None)
    refused(call, kv(), "out must", out=A + 4)
    refused(call, kv(), "out must", os=-1536)


def test_more_tiles_than_a_call_takes():
    refused(paged, kv(n_seq=65535, n_kv_heads=1024, head_stride=128, max_pages=1 << 16, table_stride=1 << 16),
            "more than one call", heads=1024, qs=131072, os=131072)


def test_workspace_too_small_or_misaligned():
    s = kv()
    need = lib().qwen_select_pages_workspace(ctypes.byref(s))
    assert need >= 3 * 2 * 8 * 8
    refused(select, s, "workspace", bytes=need - 1)
    refused(select, s, "workspace", ws=A + 16)
    refused(select, s, "workspace", ws=None)


def test_append_arguments():
    refused(append, kv(), "rot_dim", rot=0)
    refused(append, kv(), "rot_dim", rot=24)
    refused(append, kv(), "rot_dim", rot=144)
    refused(append, kv(), "inv_freq", inv=None)
    refused(append, kv(), "n_tokens", n=4)
    refused(append, kv(), "null k", k=None)
    refused(append, kv(), "null v", v=None)
    refused(append, kv(), "null q_out", out=None)
    refused(append, kv(), "k must", ks=248)
    refused(append, kv(), "v must", vs=260)


def test_selection_arguments():
    refused(select, kv(bounds=None), "bounds")
    refused(select, kv(), "n_select", n=0)
    refused(select, kv(), "n_select", n=3, first=2, last=2)
    refused(select, kv(), "n_select", n=4, first=0xFFFFFFFF, last=1)
    refused(select, kv(), "pages", pages=None)
    refused(sparse, kv(), "pages", pages=None)
    refused(sparse, kv(), "n_select", n=0)


def test_prefix_arguments():
    refused(prefix, kv(), "prefix_pages", pages=None)
    refused(prefix, kv(), "prefix_len", len=(1 << 24) + 1)


def test_no_sequences_is_nothing_to_do():
    for call in (paged, prefix, select, sparse):   # an empty tensor's address is null
        assert call(kv(n_seq=0, page_table=None), q=None) == _lib.QWEN_OK
    assert append(kv(n_seq=0, page_table=None), n=0, q=None, k=None, v=None, out=None) == _lib.QWEN_OK
    assert append(kv(), n=0, cu=A, q=None, k=None, v=None, out=None) == _lib.QWEN_OK


@pytest.mark.parametrize("fields,heads,length", [
    (dict(n_seq=0), 12, 100), (dict(n_seq=0xFFFFFFFF), 12, 100), (dict(n_kv_heads=0), 12, 100), (dict(), 0, 100),
    (dict(), 13, 100), (dict(), 0xFFFFFFFE, 100), (dict(n_kv_heads=0xFFFFFFFF), 0xFFFFFFFF, 100),
    (dict(max_pages=0xFFFFFFFF), 12, 100)])
def test_no_workspace_for_what_is_refused(fields, heads, length):
    s = ctypes.byref(kv(**fields))
    assert lib().qwen_attention_paged_workspace(s, heads) == 0
    assert lib().qwen_attention_prefix_paged_workspace(s, heads, length) == 0
    assert lib().qwen_attention_sparse_paged_workspace(s, heads, 4) == 0


def test_workspace_queries():
    s = ctypes.byref(kv())
    assert lib().qwen_attention_prefix_paged_workspace(s, 12, 0xFFFFFFFF) == 0
    own = lib().qwen_attention_paged_workspace(s, 12)
    assert 0 < own == lib().qwen_attention_prefix_paged_workspace(s, 12, 0)
    assert own < lib().qwen_attention_prefix_paged_workspace(s, 12, 1 << 24)
    assert lib().qwen_select_pages_workspace(s) == 3 * 2 * 8 * 8
    for q in (lib().qwen_attention_paged_workspace, lib().qwen_attention_sparse_paged_workspace,
              lib().qwen_attention_prefix_paged_workspace, lib().qwen_select_pages_workspace):
        assert q(None, *[12, 4][:len(q.argtypes) - 1]) == 0
    assert lib().qwen_select_pages_workspace(ctypes.byref(kv(n_kv_heads=0))) == 0


def test_python_handle_is_packed_as_the_struct_is_laid_out():
    from qweninferenceengine_b200 import ops

    values = list(range(1, 16))
    packed = PagedKVStruct.from_buffer_copy(ops._PAGED_KV.pack(*values))
    assert [getattr(packed, f) for f, _ in PagedKVStruct._fields_] == values


def test_python_handle_wants_device_tensors():
    import torch

    from qweninferenceengine_b200 import ops

    k = torch.zeros((4, 16, 2, 128), dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.PagedKV(k, k, torch.zeros((1, 4), dtype=torch.int32))
