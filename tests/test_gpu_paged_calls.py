"""Calls of the paged-cache wrappers that the documents allow and nothing else tests."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import paged_reference as ref  # noqa: E402
from qweninferenceengine_b200 import ops  # noqa: E402
from qweninferenceengine_b200._lib import QWEN_OK, lib  # noqa: E402

F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(autouse=True)
def clean_status(cuda):
    yield
    assert lib().qwen_ops_status(torch.cuda.current_stream().cuda_stream) == QWEN_OK


def test_a_batch_that_ran_empty():
    c = ref.Cache(1, [20], 12, 2, 128, 16, F16, prefix=20)
    c.make_bounds()
    kv = ops.PagedKV(c.k, c.v, c.table[:0], c.bounds)
    q, lens, x = c.q[:0], c.seq_len[:0], c.randn(1, 16, 128)[:0]
    inv = torch.ones(64, device="cuda")
    before = c.k.clone()
    assert ops.rope_append_paged(kv, x[:, :12], x[:, 12:14], x[:, 14:], lens, inv).shape == (0, 12, 128)
    pages = ops.select_pages(kv, q, lens, 3)
    assert pages.shape == (0, 2, 3)
    for out, lse in (ops.attention_paged(kv, q, lens, return_lse=True),
                     ops.attention_prefix_paged(kv, q, lens, c.prefix_pages, 20, return_lse=True),
                     ops.attention_sparse_paged(kv, q, lens, pages, return_lse=True)):
        assert out.shape == (0, 12, 128) and lse.shape == (0, 12)
    assert torch.equal(torch.nan_to_num(c.k), torch.nan_to_num(before))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H,K,D", [(12, 2, 128), (34, 2, 64)])
@pytest.mark.parametrize("prefix", [0, 200])
def test_infinite_values_show_as_what_they_are(dtype, H, K, D, prefix):
    """An infinite value of a position that counts gives that infinity in its element of
    the heads that read it, and leaves the others alone; behind the last position it does
    not count."""
    c = ref.Cache(2, [1, 40, 130, 300], H, K, D, 64, dtype, prefix=prefix)
    want = ref.attention(c, D ** -0.5)
    G = H // K
    c.v[int(c.table[0, 0]), 0, 1, 5] = float("inf")
    c.v[int(c.table[1, 0]), 39, 0, 7] = float("-inf")
    c.v[int(c.table[1, 0]), 40] = float("inf")
    c.v[int(c.table[2, 2]), 1, 1, 63] = float("inf")
    c.v[int(c.table[3, 1]), 3, 0, 0] = float("inf")
    c.v[int(c.table[3, 4]), 43, 0, 1] = float("-inf")
    there = torch.zeros((4, H, D), device="cuda")
    there[0, G:, 5], there[1, :G, 7], there[2, G:, 63], there[3, :G, 0], there[3, :G, 1] = 1, -1, 1, 1, -1
    out, lse = ops.attention_prefix_paged(c.handle(), c.q, c.seq_len, c.prefix_pages, prefix, return_lse=True)
    assert torch.equal(torch.isposinf(out), there == 1) and torch.equal(torch.isneginf(out), there == -1)
    out = torch.where(there == 0, out, want[0].to(dtype))
    ref.assert_attention((out, lse), want)
