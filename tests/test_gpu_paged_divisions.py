"""The paged-cache operators at the sizes from which their work is divided another way,
against their formulas in 64 bits (paged_reference.py derives the tolerances)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import paged_batch_reference  # noqa: E402
import paged_reference as ref  # noqa: E402
from test_gpu_paged import check_append  # noqa: E402
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


# ---------------------------------------------------------------- selection --
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("S", [2, 500, 8195, 9000])
def test_select_more_pages_than_shared_memory_holds(dtype, S):
    """Lists that compete among more than 8192 pages."""
    c = ref.Cache(S, [16 * 9500 - 3, 16 * 8196, 16 * 8195, 40], 4, 2, 64, 16, dtype)
    c.make_bounds()
    pages = ops.select_pages(c.handle(), c.q, c.seq_len, S, n_first=1, n_last=1)
    assert torch.equal(pages.cpu(), ref.select(c, S, 1, 1))


@pytest.mark.parametrize("levels", [1, 3])
def test_select_ties_among_more_pages_than_shared_memory_holds(levels):
    c = ref.Cache(40 + levels, [16 * 9000], 4, 2, 64, 16, F16)
    c.make_bounds()
    kinds = c.randn(levels, 2, 2, 64)
    kinds = torch.stack((kinds.amin(1), kinds.amax(1)), dim=1)
    c.bounds[c.table[0].long()] = kinds[torch.randint(0, levels, (9000,), generator=c.g, device="cuda")]
    for S in (3, 4000, 8999):
        assert torch.equal(ops.select_pages(c.handle(), c.q, c.seq_len, S).cpu(), ref.select(c, S, 1, 1))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [33, 41, 300])
def test_select_in_batches_of_many_sequences(dtype, n):
    """More sequences than a warp has lanes; empty and short ones between."""
    lens = [(0, 1, 16 * 5, 16 * 40 + 7, 16 * 9)[i % 5] if i % 7 else 16 * 60 for i in range(n)]
    c = ref.Cache(n, lens, 14, 2, 64, 16, dtype)
    c.make_bounds()
    kv = c.handle()
    pages = ops.select_pages(kv, c.q, c.seq_len, 6)
    assert torch.equal(pages.cpu(), ref.select(c, 6, 1, 1))
    got = ops.attention_sparse_paged(kv, c.q, c.seq_len, pages, return_lse=True)
    ref.assert_attention(got, ref.attention(c, 64 ** -0.5, lists=pages))


# ------------------------------------------------------------------- append --
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,H,K,D,P,rot,inter", [(256, 12, 2, 128, 16, 128, False), (257, 12, 2, 128, 64, 128, False),
                                                 (300, 8, 8, 64, 32, 32, True), (270, 14, 2, 64, 64, 64, False)])
def test_append_rows_of_many_sequences(dtype, n, H, K, D, P, rot, inter):
    """Beside and beyond the 256 sequences up to which rows find theirs by counting; some
    with nothing new, the first and the last among them."""
    new = [0 if i in (0, n - 1) or i % 4 == 1 else (1, 3, 17, P + 2)[i % 4] for i in range(n)]
    lens = [x + (i * 13) % (2 * P) for i, x in enumerate(new)]
    check_append(ref.Cache(n, lens, H, K, D, P, dtype), new, rot, inter, ragged=True, pad=3)


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_one_token_of_many_sequences(dtype):
    lens = [(i * 13) % 130 for i in range(400)]
    check_append(ref.Cache(9, lens, 12, 2, 128, 64, dtype), [min(x, 1) for x in lens], 128, False, ragged=False)
