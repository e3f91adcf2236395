"""The reference for whole batches says what the one for single sequences says (no GPU)."""
import pytest
import torch

import paged_batch_reference
import paged_reference as ref


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("prefix", [0, 1, 100])
def test_same_values_and_bounds(dtype, prefix):
    c = ref.Cache(prefix, [0, 1, 33, 0, 50], 6, 2, 64, 16, dtype, prefix=prefix, device="cpu")
    for one, all_ in zip(ref.attention(c, 0.2), paged_batch_reference.attention(c, 0.2)):
        finite = torch.isfinite(one)
        assert torch.equal(finite, torch.isfinite(all_))
        assert torch.allclose(one[finite], all_[finite], rtol=1e-10, atol=1e-12)
