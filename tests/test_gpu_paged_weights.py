"""Attention over pages keeps its weights to twice the type's digits, as
attention_decode_batched does: outputs that nearly cancel, where a weight rounded once
to the cache's type shows."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import paged_reference as ref  # noqa: E402
from qweninferenceengine_b200 import ops  # noqa: E402


def cancelling(seed, lens, H, K, D, P, dtype):
    """Keys in nearly equal pairs, values +1 and -1 in turn; small scores, so that fp32's
    own errors are far below a rounding to 16 bits."""
    c = ref.Cache(seed, lens, H, K, D, P, dtype)
    c.k[:, 1::2] = (c.k[:, 0::2].double() * 1.01).to(dtype)
    c.v[:, 0::2], c.v[:, 1::2] = 1.0, -1.0
    c.q *= 0.1
    return c


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,K,D,P", [(12, 2, 128, 16), (32, 8, 128, 64), (14, 2, 64, 32), (34, 2, 64, 256)])
def test_weights_are_not_rounded_to_the_type(dtype, H, K, D, P):
    """paged_reference.attention's bound with u^2 for the weights' u: the rest of a weight
    after its first rounding (u of it at most) is rounded once itself.  |v| is 1, so the
    bound's sum of p |v| is 1; outputs are rounded once (u of them)."""
    c = cancelling(5, [2 * (i + 1) for i in range(60)] + [1000, 4098], H, K, D, P, dtype)
    u = ref.U[dtype]
    want, want_lse, tol, lse_tol = ref.attention(c, D ** -0.5)
    tol = tol - u + u * u
    kv = c.handle()
    columns = torch.arange(c.width, dtype=torch.int32, device="cuda").expand(len(c.lens), K, -1).contiguous()
    for got in (ops.attention_paged(kv, c.q, c.seq_len, return_lse=True),
                ops.attention_sparse_paged(kv, c.q, c.seq_len, columns, return_lse=True)):
        ref.assert_attention(got, (want, want_lse, tol, lse_tol))
