"""Calls over a 4-bit paged cache at the edges of what the documents allow."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import paged_q4_reference as ref  # noqa: E402
from qweninferenceengine_b200 import ops  # noqa: E402
from qweninferenceengine_b200._lib import QWEN_ERR_INVALID_ARGUMENT, QWEN_OK, lib  # noqa: E402

F16, BF16 = torch.float16, torch.bfloat16
DTYPES = [F16, BF16]


def status():
    return lib().qwen_ops_status(torch.cuda.current_stream().cuda_stream)


@pytest.fixture(autouse=True)
def clean_status(cuda):
    yield
    assert status() == QWEN_OK


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("n,H,K,D", [(1, 12, 2, 128), (3, 16, 8, 64), (33, 40, 2, 64), (1000, 2, 1, 128)])
def test_every_length_beyond_the_table(n, H, K, D, kept, dtype):
    """Reported, nothing is written; the next call's lengths are served."""
    c = ref.Cache(1, [40] * n, H, K, D, 16, dtype, width=3, kept=kept)
    kv = c.handle()
    weights = c.weights.clone() if kept else None
    for length in (49, 2 ** 31 - 1, -1):
        out = torch.full((n, H, D), 7.0, dtype=dtype, device="cuda")
        ops.attention_paged_q4(kv, c.q, torch.full((n,), length, dtype=torch.int32, device="cuda"), out=out)
        assert status() == QWEN_ERR_INVALID_ARGUMENT
        assert (out == 7.0).all()
        if kept:
            assert torch.equal(c.weights, weights)
    got = ops.attention_paged_q4(kv, c.q, c.seq_len, return_lse=True)
    r = ref.attention(c, D ** -0.5)
    ref.check_attention(got, r)
    if kept:
        ref.check_weights(c.weights, weights, r)
