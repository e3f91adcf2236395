"""The paged-cache operators at the sizes from which their work is divided another way,
against their formulas in 64 bits (paged_reference.py derives the tolerances)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import paged_batch_reference  # noqa: E402
import paged_reference as ref  # noqa: E402
from qweninferenceengine_b200 import ops  # noqa: E402
from qweninferenceengine_b200._lib import QWEN_OK, lib  # noqa: E402

F16, BF16 = torch.float16, torch.bfloat16
DTYPES = [F16, BF16]


@pytest.fixture(autouse=True)
def clean_status(cuda):
    yield
    assert lib().qwen_ops_status(torch.cuda.current_stream().cuda_stream) == QWEN_OK


# ------------------------------------------------------------ shared prefix --
# Row tiles x kv heads beyond the SMs that the prefix gets: a CTA of k_prefix goes on
# from one unit's piece to the next.  Even and odd numbers of row tiles (a lone tile in
# a run), prefixes that end inside a tile, one of less than a tile, one step or many.
PREFIXES = [(256, 64, 8, 128, 128, 1000), (400, 32, 8, 128, 256, 1000), (517, 32, 8, 128, 64, 129),
            (1024, 12, 2, 128, 256, 4096), (1100, 12, 2, 128, 16, 77), (1300, 16, 8, 64, 64, 700),
            (2048, 14, 2, 64, 128, 300), (160, 64, 64, 128, 32, 515), (100, 128, 128, 64, 256, 2049)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,H,K,D,P,prefix", PREFIXES)
def test_prefix_units_beyond_the_ctas(dtype, n, H, K, D, P, prefix):
    lens = [(i * 37) % 50 if i % 3 else 0 for i in range(n)]
    c = ref.Cache(n + prefix, lens, H, K, D, P, dtype, prefix=prefix)
    kv = c.handle()
    call = lambda: ops.attention_prefix_paged(kv, c.q, c.seq_len, c.prefix_pages, prefix, return_lse=True)  # noqa: E731
    out, lse = call()
    ref.assert_attention((out, lse), paged_batch_reference.attention(c, D ** -0.5))
    for _ in range(10):
        again = call()
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)


@pytest.mark.parametrize("dtype", DTYPES)
def test_prefix_units_beyond_the_ctas_captured(dtype):
    """The same replayed over other queries, in the memory that the last replay left."""
    c = ref.Cache(7, [5, 0, 40, 1] * 100, 32, 8, 128, 64, dtype, prefix=900)
    kv = c.handle()
    ops.attention_prefix_paged(kv, c.q, c.seq_len, c.prefix_pages, 900)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = ops.attention_prefix_paged(kv, c.q, c.seq_len, c.prefix_pages, 900, return_lse=True)
    for _ in range(2):
        c.q.copy_(c.randn(400, 32, 128))
        g.replay()
        ref.assert_attention(got, paged_batch_reference.attention(c, 128 ** -0.5))
