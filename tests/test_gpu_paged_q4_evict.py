"""Eviction of rows of which a CTA has more slots than it holds keys of, or numbers at
once (16384): more rows than two an SM, or a row over more than eight times that."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import paged_q4_reference as ref  # noqa: E402
from qweninferenceengine_b200 import ops  # noqa: E402
from qweninferenceengine_b200._lib import QWEN_OK, lib  # noqa: E402

F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(autouse=True)
def clean_status(cuda):
    yield
    assert lib().qwen_ops_status(torch.cuda.current_stream().cuda_stream) == QWEN_OK


def moves(weights, positions, n_keep, n_first, n_recent):
    """(to, from) of one (sequence, kv head) of more than n_keep slots."""
    at = positions.long()
    guarded = (at < n_first) | (at > at.max() - n_recent)
    order = weights.sort(descending=True, stable=True).indices   # (NaN first)
    order = order[(~guarded)[order].to(torch.int8).sort(stable=True).indices]
    kept = torch.zeros_like(guarded)
    kept[order[:n_keep]] = True
    below = torch.arange(len(at), device=at.device) < n_keep
    return (~kept & below).nonzero()[:, 0], (kept & ~below).nonzero()[:, 0]


def check(c, n_keep, n_first, n_recent, times=4):
    """All of the cache is what the moves make of it, each time."""
    pool, w, p = c.pool.clone(), c.weights.clone(), c.positions.clone()
    want_pool, want_w, want_p = pool.clone(), w.clone(), p.clone()
    for i, x in enumerate(c.lens):
        for h in range(c.kv_heads):
            if x <= n_keep:
                continue
            to, src = moves(w[i, h, :x], p[i, h, :x], n_keep, n_first, n_recent)
            (tp, tb, tr), (sp, sb, sr) = c.place(i, to), c.place(i, src)
            for part in ref.views(want_pool, c.dim, c.dtype):
                part[tp, h, tb, :, tr] = part[sp, h, sb, :, sr]
            want_w[i, h, to], want_p[i, h, to] = w[i, h, src], p[i, h, src]
    for _ in range(times):
        c.pool.copy_(pool)
        c.weights.copy_(w)
        c.positions.copy_(p)
        got = ops.evict_paged_q4(c.handle(), c.seq_len, n_keep, n_first, n_recent)
        assert got.tolist() == [min(x, n_keep) for x in c.lens]
        assert torch.equal(c.weights.nan_to_num(-3.0), want_w.nan_to_num(-3.0))
        assert torch.equal(c.positions, want_p) and torch.equal(c.pool, want_pool)
    c.pool.copy_(pool)
    c.weights.copy_(w)
    c.positions.copy_(p)


def cache(lens, kv_heads, page=256):
    c = ref.Cache(1, [0] * len(lens), kv_heads, kv_heads, 64, page, F16, width=-(-max(lens) // page), kept=True)
    c.lens, c.seq_len = lens, torch.tensor(lens, dtype=torch.int32, device="cuda")
    c.pool.copy_(torch.randint(0, 256, c.pool.shape, generator=c.g, device="cuda", dtype=torch.uint8))
    for i, x in enumerate(lens):
        if x:
            c.positions[i, :, :x] = torch.randperm(x, generator=c.g, device="cuda").to(torch.int32)
    return c


# (a budget in the first tile, in the second, at their border, in the last)
@pytest.mark.parametrize("keep", [2047, 16384, 16385, 20000, 39990])
@pytest.mark.parametrize("lens,kv_heads", [([40000, 16384, 16385, 33000, 0, 1] + [40000] * 71, 2),
                                           ([150000, 131072], 1)])
def test_rows_of_several_tiles(lens, kv_heads, keep):
    c = cache(lens, kv_heads)
    check(c, keep, 4, keep // 4)   # weights that differ: no ties to number
    c.weights.copy_((c.weights * 4).floor())
    c.weights[:, :, 5::97] = math.nan
    c.weights[:, :, 6::97] = -math.inf
    check(c, keep, 4, keep // 4, times=1)
    check(c, keep, 0, 0, times=1)
    check(c, keep, keep + 100, 0, times=1)   # more guarded slots than stay
    c.weights.fill_(1.0)
    check(c, keep, 0, 3, times=1)
