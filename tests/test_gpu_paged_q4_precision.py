"""What decode attention over a 4-bit paged cache must not lose: weights, codes and sums
where the bounds of test_gpu_paged_q4.py, which grow with the length, are wide."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import paged_q4_reference as ref  # noqa: E402
from paged_reference import U  # noqa: E402
from qweninferenceengine_b200 import ops  # noqa: E402
from qweninferenceengine_b200._lib import QWEN_OK, lib  # noqa: E402

F16, BF16 = torch.float16, torch.bfloat16
DTYPES = [F16, BF16]


@pytest.fixture(autouse=True)
def clean_status(cuda):
    yield
    assert lib().qwen_ops_status(torch.cuda.current_stream().cuda_stream) == QWEN_OK


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,H,K,D,P", [([1000], 12, 2, 128, 64), ([16, 70, 1777], 16, 8, 64, 16),
                                          ([4096] * 9, 40, 2, 128, 256)])
def test_attention_of_elements_that_are_zero(dtype, lens, H, K, D, P):
    """An element that is 0 in every slot, the least of its groups, has code 0 and low 0 whatever
    the groups' steps: products with it are 0, and so is the output, exactly."""
    c = ref.Cache(1, [0] * len(lens), H, K, D, P, dtype, width=-(-max(lens) // P))
    c.lens, c.seq_len = lens, torch.tensor(lens, dtype=torch.int32, device="cuda")
    zero = torch.ones(D, dtype=torch.bool, device="cuda")
    zero[5::32] = False
    for i, x in enumerate(lens):
        v = c.randn(x, K, D).abs()
        v[..., zero] = 0
        c.store(i, c.all_slots(i), c.randn(x, K, D), v)
    out = ops.attention_paged_q4(c.handle(), c.q, c.seq_len)
    assert (out[..., zero] == 0).all()
    assert (out[..., ~zero] > 0).all()


def test_attention_of_long_bf16_contexts_is_not_off_to_one_side():
    """The mean error over a sequence's outputs near zero, whose parts (lows, steps times codes)
    are not.

    A tile's MMAs (four for lows, four for codes) cut off at most 2^-23 of their sums each:
    together 2^-20 A of A = sum of weights (|low| + 15 step).  All else errs to both sides: the
    output's rounding, u |out| at most, weights of 16 bits, 2^-17 A at most each and, as their
    errors are independent, 2^-17 A / sqrt(L / 16) in the sum of L slots whose weights, over
    L / 16, differ little, and the additions of the T tiles, 2^-24 A each.  The mean of N outputs'
    errors is within 6 of its deviations."""
    n, L, H, K, D = 12, 16384, 32, 8, 128
    c = ref.Cache(50, [L] * n, H, K, D, 64, BF16)
    out = ops.attention_paged_q4(c.handle(), c.q, c.seq_len)[3].double()
    slots = c.all_slots(3)
    k, v = c.rows(3, slots)
    page, block, r = c.place(3, slots)
    step, low = ref.views(c.pool, D, BF16)[3][page, :, block, :, r].double().abs().unbind(-1)
    want, size = [], []
    for h in range(K):
        w = torch.softmax(c.q[3, h * 4: h * 4 + 4].double() @ k[:, h].T * D ** -0.5, -1)
        want.append(w @ v[:, h])
        size.append((w @ (low + 15 * step)[:, h]).amax())
    want, A = torch.cat(want), torch.stack(size).amax().item()
    off = (out - want).mean().abs().item()
    each = U[BF16] ** 2 * want.pow(2).mean().item() + (2.0 ** -34 * 16 / L + L / 128 * 2.0 ** -48) * A ** 2
    assert off <= 2.0 ** -20 * A + 6 * (each / want.numel()) ** 0.5, (off, A)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,L,H,K,D", [(1, 16384, 12, 2, 128), (8, 16384, 32, 8, 128), (3, 20011, 16, 8, 64)])
@pytest.mark.parametrize("above", [10.0, 18.0, 20.0])
@pytest.mark.parametrize("alike", [False, True])
def test_attention_beside_a_heavy_slot(dtype, n, L, H, K, D, above, alike):
    """One slot of a score `above` the others' and a value near zero, as the first tokens of a
    text have: the output is what the many others add up to, each of a weight of e^-above.

    Bounds: scores are off by d as in paged_q4_reference.py, all weights alike (2 d, relative
    to the sum that each is divided by); a weight with its step and low 2^-16 of them; sums of
    T tiles, over up to 32 pieces, at random to both sides, at most (2^-20 + 6 2^-24 sqrt(T))
    of what is summed, B = sum of weights (|low| + 15 step); and the output's rounding."""
    c = ref.Cache(51, [0] * n, H, K, D, 64, dtype, width=L // 64 + 1)
    c.lens, c.seq_len = [L] * n, torch.full((n,), L, dtype=torch.int32, device="cuda")
    slots = c.all_slots(0)
    for i in range(n):
        k, v = c.randn(L, K, D) * 0.02, c.randn(L, K, D)
        if alike:
            k = k[:1].expand(L, -1, -1).clone()
        k[7], v[7] = above * D ** -0.5, v[7] * 2.0 ** -13
        c.store(i, slots, k, v)
    c.q = (1 + 0.01 * c.randn(n, H, D).double()).to(dtype)
    out = ops.attention_paged_q4(c.handle(), c.q, c.seq_len)[0].double()
    k, v = c.rows(0, slots)
    ka = c.sizes(0, slots)[0]
    page, block, r = c.place(0, slots)
    step, low = ref.views(c.pool, D, dtype)[3][page, :, block, :, r].double().abs().unbind(-1)
    G = H // K
    for h in range(K):
        x = c.q[0, h * G: (h + 1) * G].double()
        s = x @ k[:, h].T * D ** -0.5
        d = 2.0 ** -23 * (2 * D * (x.abs() @ ka[:, h].T * D ** -0.5).amax() + 16 + 2 * s.abs().amax())
        w = torch.softmax(s, -1)
        want = w @ v[:, h]
        B = (w @ (low + 15 * step)[:, h]).repeat_interleave(32, -1)
        tol = B * (2 * d + 2.0 ** -16 + 2.0 ** -20 + 6 * 2.0 ** -24 * (L / 128) ** 0.5) + U[dtype] * want.abs() + 2.0 ** -25
        off = (out[h * G: (h + 1) * G] - want).abs() - tol
        assert off.max().item() <= 0, (off.max().item(), tol.max().item(), want.abs().max().item())


@pytest.mark.parametrize("big,grow", [(6e33, 0.0), (6e30, 5.0)])
def test_attention_of_bf16_values_near_the_types_end(big, grow):
    """Length times value 10^35, with scores that grow, so that weights pass those that a run
    began with (they are below 2^8); and 10^38 with scores around one value, whose weights stay
    about 1: 2 10^38 is the most that their sums come to.  So many sequences that one run
    has a whole one."""
    n, L, H, K, D = 128, 16384, 16, 8, 64
    c = ref.Cache(60, [0] * n, H, K, D, 64, BF16, width=L // 64)
    c.lens, c.seq_len = [L] * n, torch.full((n,), L, dtype=torch.int32, device="cuda")
    c.pool.copy_(torch.randint(0, 256, (1, *c.pool.shape[1:]), generator=c.g, device="cuda", dtype=torch.uint8))
    _, _, ks, vs = ref.views(c.pool, D, BF16)
    vs[..., 0], vs[..., 1] = 2 * big / 15, -big
    ks[..., 0] = 2.0 ** -6
    for i in range(n):   # every element of a slot's key alike, but for its codes
        page, block, r = c.place(i, c.all_slots(i))
        ks[page, :, block, :, r, 1] = (torch.arange(L, device="cuda") * (grow * D ** -0.5 / L)).to(BF16)[:, None, None]
    c.q = (1 + 0.01 * c.randn(n, H, D).double()).to(BF16)
    got = ops.attention_paged_q4(c.handle(), c.q, c.seq_len, return_lse=True)
    assert torch.isfinite(got[0]).all() and torch.isfinite(got[1]).all()
    for i in (0, n - 1):
        only = [L if j == i else 0 for j in range(n)]
        want = ref.attention(c, D ** -0.5, lens=only)
        ref.check_attention(tuple(x[i: i + 1] for x in got), tuple(x[i: i + 1] for x in want))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,K,D", [(12, 2, 128), (16, 8, 64)])
def test_attention_of_one_slot_is_its_value(dtype, H, K, D):
    """A weight of 1 and a sum of 1: low + code step, formed in fp32 and rounded to the type."""
    n = 400
    c = ref.Cache(70, [1] * n, H, K, D, 16, dtype)
    _, vc, _, vs = ref.views(c.pool, D, dtype)
    vc.copy_(torch.randint(0, 256, vc.shape, generator=c.g, device="cuda", dtype=torch.uint8))
    scale = 2.0 ** torch.randint(-8, 9, vs.shape[:-1], generator=c.g, device="cuda")
    vs[..., 0] = (torch.rand(vs.shape[:-1], generator=c.g, device="cuda") * scale).to(dtype)
    vs[..., 1] = (torch.randn(vs.shape[:-1], generator=c.g, device="cuda") * scale).to(dtype)
    out = ops.attention_paged_q4(c.handle(), c.q, c.seq_len)
    page = c.table[:, 0].long()
    code = torch.stack((vc[page, :, 0, :, 0] & 15, vc[page, :, 0, :, 0] >> 4), -1).flatten(-2)
    assert code.unique().numel() == 16
    p = vs[page, :, 0, :, 0].float()
    want = (p[..., 1:] + code.float() * p[..., :1]).flatten(-2).to(dtype)   # (the product is exact)
    assert torch.equal(out, want.repeat_interleave(H // K, 1))
