"""Arguments that the entry points over a 4-bit cache refuse before they touch a device
(runs without a GPU): the buffers are made-up addresses that nothing reads."""
import ctypes

import pytest

from qweninferenceengine_b200 import _lib
from qweninferenceengine_b200._lib import QWEN_ERR_INVALID_ARGUMENT, QWEN_OK, PagedKVQ4Struct, lib

A = 0x10000   # a 256-byte aligned address


def kv(**fields):
    s = PagedKVQ4Struct(A, A, A, A, 2 * 2560, 2560, 64, 16, 2, 128, 3, 8, 8, _lib.QWEN_DTYPE_F16)
    for name, value in fields.items():
        setattr(s, name, value)
    return s


def append(s, **o):
    a = dict(q=A, qs=1536, k=A, ks=256, v=A, vs=256, out=A, os=1536, heads=12, n=3, lens=A, cu=None, pos=A,
             ps=3, axes=1, which=None, inv=A, rot=128, inter=0) | o
    return lib().qwen_rope_append_paged_q4(
        ctypes.byref(s) if s else None, a["q"], a["qs"], a["k"], a["ks"], a["v"], a["vs"], a["out"], a["os"],
        a["heads"], a["n"], a["lens"], a["cu"], a["pos"], a["ps"], a["axes"], a["which"], a["inv"], a["rot"],
        a["inter"], None)


def attend(s, **o):
    a = dict(q=A, qs=1536, out=A + (1 << 20), os=1536, lse=None, heads=12, lens=A, ws=A, bytes=1 << 40) | o
    return lib().qwen_attention_paged_q4(ctypes.byref(s) if s else None, a["q"], a["qs"], a["out"], a["os"],
                                         a["lse"], a["heads"], a["lens"], 0.1, a["ws"], a["bytes"], None)


def expand(s, **o):
    a = dict(lens=A, cu=None, n=3, k=A, ks=256, v=A, vs=256) | o
    return lib().qwen_expand_paged_q4(ctypes.byref(s) if s else None, a["lens"], a["cu"], a["n"], a["k"],
                                      a["ks"], a["v"], a["vs"], None)


def evict(s, **o):
    a = dict(lens=A, keep=10, first=1, recent=1, out=A, ws=A, bytes=1 << 40) | o
    return lib().qwen_evict_paged_q4(ctypes.byref(s) if s else None, a["lens"], a["keep"], a["first"],
                                     a["recent"], a["out"], a["ws"], a["bytes"], None)


OPS = [append, attend, expand, evict]


def refused(call, s, text, **o):
    assert call(s, **o) == QWEN_ERR_INVALID_ARGUMENT
    assert text in lib().qwen_last_error().decode()


@pytest.mark.parametrize("call", OPS)
@pytest.mark.parametrize("fields,text", [
    (dict(pool=None), "null cache"), (dict(page_table=None), "null cache"), (dict(dtype=2), "dtype"),
    (dict(head_dim=96), "head_dim"), (dict(page_size=8), "page_size"), (dict(page_size=48), "page_size"),
    (dict(page_size=512), "page_size"), (dict(n_pages=0), "n_pages"), (dict(n_seq=65536), "n_seq"),
    (dict(max_pages=0), "max_pages"), (dict(max_pages=1 << 21, table_stride=1 << 21), "max_pages"),
    (dict(table_stride=7), "table_stride"), (dict(n_kv_heads=0), "n_heads"), (dict(n_kv_heads=1025), "n_heads"),
    (dict(page_stride=0), "stride"), (dict(head_stride=-16), "stride"), (dict(head_stride=2568), "stride"),
    (dict(pool=A + 8), "aligned"), (dict(weights=A + 4), "aligned"), (dict(positions=A + 8), "aligned")])
def test_cache_descriptions(call, fields, text):
    refused(call, kv(**fields), text)


def test_null_and_empty():
    for call in OPS:
        refused(call, None, "null kv")
    for call, o in ((append, dict(n=0)), (attend, {}), (expand, dict(n=0)), (evict, {})):
        assert call(kv(n_seq=0, page_table=None), **o) == QWEN_OK


def test_append_arguments():
    refused(append, kv(), "null q", q=None)
    refused(append, kv(), "null k", k=None)
    refused(append, kv(), "null v", v=None)
    refused(append, kv(), "null q_out", out=None)
    refused(append, kv(), "q must", qs=1528)
    refused(append, kv(), "k must", ks=252)
    refused(append, kv(), "v must", v=A + 2)
    refused(append, kv(), "seq_len", lens=None)
    refused(append, kv(), "inv_freq", inv=None)
    refused(append, kv(), "rot_dim", rot=24)
    refused(append, kv(), "rot_dim", rot=144)
    refused(append, kv(), "rot_dim", rot=0)
    refused(append, kv(), "n_heads", heads=13)
    refused(append, kv(), "n_tokens", n=4)
    refused(append, kv(), "n_tokens", n=(1 << 24) + 1, cu=A)
    refused(append, kv(), "n_axes", axes=0)
    refused(append, kv(), "n_axes", axes=5, which=A)
    refused(append, kv(), "n_axes", axes=2)
    refused(append, kv(), "n_axes", axes=2, which=A, pos=None)
    refused(append, kv(), "position_stride", axes=2, which=A, ps=-8)
    refused(append, kv(), "position_stride", axes=2, which=A, ps=1 << 38)
    refused(append, kv(n_kv_heads=1024), "n_tokens", heads=1024, qs=1 << 17, os=1 << 17, ks=1 << 17, vs=1 << 17,
            n=1 << 23, cu=A)


def test_attention_arguments():
    refused(attend, kv(), "null q", q=None)
    refused(attend, kv(), "null out", out=None)
    refused(attend, kv(), "out must be", out=A + (1 << 20) + 8)
    refused(attend, kv(), "seq_len", lens=None)
    refused(attend, kv(), "n_heads", heads=130)
    s = kv()
    need = lib().qwen_attention_paged_q4_workspace(ctypes.byref(s), 12)
    assert need > 0
    refused(attend, s, "workspace", bytes=need - 1)
    refused(attend, s, "workspace", ws=A + 16)
    refused(attend, s, "workspace", ws=None)


def test_expand_arguments():
    refused(expand, kv(), "null k", k=None)
    refused(expand, kv(), "v must", vs=248)
    refused(expand, kv(), "seq_len", lens=None)
    refused(expand, kv(), "n_rows", n=4)
    refused(expand, kv(), "n_rows", n=(1 << 30) + 1, cu=A)


def test_evict_arguments():
    refused(evict, kv(weights=None), "weights")
    refused(evict, kv(positions=None), "weights")
    refused(evict, kv(), "null seq_len", lens=None)
    refused(evict, kv(), "new_len", out=None)
    refused(evict, kv(), "n_keep", keep=0)
    refused(evict, kv(), "n_keep", keep=(1 << 24) + 1)
    refused(evict, kv(), "n_first", first=(1 << 30) + 1)
    refused(evict, kv(), "n_recent", recent=(1 << 30) + 1)
    s = kv()
    need = lib().qwen_evict_paged_q4_workspace(ctypes.byref(s), 10)
    assert need > 0
    refused(evict, s, "workspace", bytes=need - 1)
    refused(evict, s, "workspace", ws=A + 16)


def test_workspace_of_refused_sizes_is_none():
    for fields in (dict(head_dim=96), dict(dtype=7), dict(page_size=8), dict(n_seq=0), dict(n_kv_heads=5)):
        assert lib().qwen_attention_paged_q4_workspace(ctypes.byref(kv(**fields)), 12) == 0
    for fields in (dict(head_dim=96), dict(dtype=7), dict(page_size=8), dict(n_seq=0)):
        assert lib().qwen_evict_paged_q4_workspace(ctypes.byref(kv(**fields)), 10) == 0
    assert lib().qwen_evict_paged_q4_workspace(ctypes.byref(kv()), 0) == 0
    assert lib().qwen_evict_paged_q4_workspace(None, 10) == 0
