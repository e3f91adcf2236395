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
