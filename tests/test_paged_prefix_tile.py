"""k_prefix: the bytes of a stream's query tile, from the kernel's own arithmetic
(qwen_paged_prefix_tile).  At the end of a piece each softmax warp stages its output
rows in the tile, and then, without waiting for the others, writes its rows of the next
piece's queries there: no warp may touch what another one stages."""
import ctypes

import pytest

from qweninferenceengine_b200 import _lib


@pytest.mark.parametrize("dim", [64, 128])
def test_a_warp_stages_where_only_its_own_queries_go(dim):
    hook = ctypes.CDLL(_lib.LIB_PATH).qwen_paged_prefix_tile
    n_query, n_stage = 16 * dim // 8, 32 * dim // 16
    query, stage = (ctypes.c_int * (8 * n_query))(), (ctypes.c_int * (8 * n_stage))()
    hook(ctypes.c_int(dim), query, stage)
    written = [list(query[j * n_query:(j + 1) * n_query]) for j in range(8)]
    staged = [list(stage[j * n_stage:(j + 1) * n_stage]) for j in range(8)]
    whole = set(range(0, 128 * dim * 2, 16))
    for chunks in (written, staged):
        assert sorted(x for w in chunks for x in w) == sorted(whole)   # each chunk once
    for j in range(8):
        for other in range(8):
            if other != j:
                assert not set(staged[j]) & set(written[other]), (j, other)
