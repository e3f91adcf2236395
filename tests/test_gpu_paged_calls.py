"""Calls of the paged-cache wrappers that the documents allow and nothing else tests."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import paged_batch_reference  # noqa: E402
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


class Batch:
    """A cache of many short sequences, made at once (ref.Cache fills page by page)."""

    def __init__(self, seed, lens, H, K, D, P, dtype, prefix):
        g = torch.Generator(device="cuda").manual_seed(seed)
        n = len(lens)
        self.dtype, self.kv_heads, self.page, self.prefix = dtype, K, P, prefix
        self.width = -(-max(lens) // P)
        n_prefix = -(-prefix // P)
        n_pages = n * self.width + n_prefix
        order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
        self.table, self.prefix_pages = order[: n * self.width].view(n, self.width), order[n * self.width:].clone()
        self.k, self.v = (torch.randn((n_pages, P, K, D), generator=g, device="cuda").to(dtype) for _ in range(2))
        self.q = torch.randn((n, H, D), generator=g, device="cuda").to(dtype)
        self.seq_len = torch.tensor(lens, dtype=torch.int32, device="cuda")


def test_as_many_sequences_as_a_call_takes():
    n, H, K, D, P = 65535, 4, 1, 64, 16
    c = Batch(3, [(i * 7) % 21 for i in range(n)], H, K, D, P, F16, 150)
    kv = ops.PagedKV(c.k, c.v, c.table)
    got = ops.attention_prefix_paged(kv, c.q, c.seq_len, c.prefix_pages, 150, return_lse=True)
    ref.assert_attention(got, paged_batch_reference.attention(c, D ** -0.5))
    c.prefix = 0
    want = paged_batch_reference.attention(c, D ** -0.5)
    ref.assert_attention(ops.attention_paged(kv, c.q, c.seq_len, return_lse=True), want)
    # bounds of all slots, also of those that hold nothing: any bounds do for a list of all pages
    kv = ops.PagedKV(c.k, c.v, c.table, torch.stack((c.k.amin(1), c.k.amax(1)), dim=1))
    pages = ops.select_pages(kv, c.q, c.seq_len, 2)
    have = (c.seq_len + P - 1) // P
    at = torch.arange(2, device="cuda")
    assert torch.equal(pages[:, 0], torch.where(at < have[:, None], at, -1).int())
    ref.assert_attention(ops.attention_sparse_paged(kv, c.q, c.seq_len, pages, return_lse=True), want)
    # one new row for every fifth sequence (of a length other than 0)
    new = (torch.arange(n, device="cuda") % 5 == 0) & (c.seq_len > 0)
    cu = torch.cat((torch.zeros(1, device="cuda"), new.cumsum(0))).to(torch.int32)
    rows, inv = int(cu[-1]), torch.full((D // 2,), 0.25, device="cuda")
    x = torch.randn((rows, H + 2 * K, D), device="cuda").to(F16)
    v0, last = c.v.clone(), c.seq_len[new].long() - 1
    page = c.table[new].gather(1, (last // P)[:, None])[:, 0].long()
    q = ops.rope_append_paged(kv, x[:, :H], x[:, H:H + K], x[:, H + K:], c.seq_len, inv, cu_tokens=cu)
    v0[page, last % P] = x[:, H + K:]
    assert torch.equal(c.v, v0)
    for got, src in ((q, x[:, :H]), (c.k[page, last % P], x[:, H:H + K])):
        y, e = ref.rotate(src, last, inv, False)
        assert ((got.double() - y).abs() - (ref.U[F16] * y.abs() + 2 * e + 1e-7)).max().item() <= 0


@pytest.mark.parametrize("n,H,K,D,P,prefix", [(3, 1, 1, 64, 16, 0), (1, 5, 1, 128, 256, 7), (2, 3, 3, 64, 32, 40)])
def test_pools_of_few_pages(n, H, K, D, P, prefix):
    """One kv head, or one page: strides of axes of one element say nothing."""
    c = ref.Cache(6, [1] * n if prefix == 0 else [P - 1] * n, H, K, D, P, BF16, prefix=prefix, spare=0)
    odd = lambda x: x.as_strided(x.shape, (x.stride(0) if x.shape[0] > 1 else 5, x.stride(1),  # noqa: E731
                                          x.stride(2) if K > 1 else 3, 1))
    kv = ops.PagedKV(odd(c.k), odd(c.v), c.table)
    lens = c.seq_len.view(torch.uint32)
    got = ops.attention_prefix_paged(kv, c.q, lens, c.prefix_pages, prefix, return_lse=True)
    ref.assert_attention(got, ref.attention(c, D ** -0.5))


def test_strided_outputs():
    c = ref.Cache(8, [100, 1, 64], 12, 2, 128, 32, F16, prefix=90)
    c.make_bounds()
    kv, inv = c.handle(), torch.full((64,), 0.25, device="cuda")
    pages = ops.select_pages(kv, c.q, c.seq_len, 4)
    x = c.randn(3, 16, 128)
    for call in (lambda o: ops.attention_prefix_paged(kv, c.q, c.seq_len, c.prefix_pages, 90, out=o),
                 lambda o: ops.attention_sparse_paged(kv, c.q, c.seq_len, pages, out=o),
                 lambda o: ops.rope_append_paged(kv, x[:, :12], x[:, 12:14], x[:, 14:], c.seq_len, inv, out=o)):
        dense = call(torch.empty_like(c.q))
        wide = torch.full((3, 14, 128), 7.0, dtype=F16, device="cuda")
        assert torch.equal(call(wide[:, 1:13]), dense)
        assert (wide[:, 0] == 7).all() and (wide[:, 13] == 7).all()


def test_captured_between_copies_and_other_streams():
    """Calls whose predecessor in the graph is a memset, a copy or another stream's kernel."""
    c = ref.Cache(9, [300, 47, 16, 129], 12, 2, 128, 16, F16, prefix=333)
    kv, q = c.handle(), torch.empty_like(c.q)
    buf, side = torch.empty(1 << 20, device="cuda"), torch.cuda.Stream()
    ops.attention_prefix_paged(kv, c.q, c.seq_len, c.prefix_pages, 333)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            q.copy_(c.q)
            dense = ops.attention_paged(kv, q, c.seq_len, return_lse=True)
        buf.zero_()
        first = ops.attention_prefix_paged(kv, c.q, c.seq_len, c.prefix_pages, 333, return_lse=True)
        main.wait_stream(side)
        second = ops.attention_prefix_paged(kv, q, c.seq_len, c.prefix_pages, 333, return_lse=True)
    for _ in range(3):
        c.q.copy_(c.randn(4, 12, 128))
        q.fill_(float("nan"))
        g.replay()
        c.prefix = 333
        want = ref.attention(c, 128 ** -0.5)
        ref.assert_attention(first, want)
        ref.assert_attention(second, want)
        c.prefix = 0
        ref.assert_attention(dense, ref.attention(c, 128 ** -0.5))


@pytest.mark.parametrize("ragged", [False, True])
def test_a_nan_key_marks_its_page(ragged):
    """Its bounds are NaN in that element (and in the one it is rotated with), and the page
    comes first in a selection."""
    c = ref.Cache(10, [16 * 40], 4, 2, 64, 16, BF16)
    c.make_bounds()
    kv, inv = c.handle(), torch.zeros(8, device="cuda")
    x = c.randn(1, 8, 64)
    x[0, 4, 3], x[0, 5, 40] = float("nan"), float("nan")
    cu = torch.tensor([0, 1], dtype=torch.int32, device="cuda") if ragged else None
    at = c.seq_len.clone().fill_(16 * 20 + 9)
    ops.rope_append_paged(kv, x[:, :4], x[:, 4:6], x[:, 6:], at, inv, cu_tokens=cu)
    b = c.bounds[int(c.table[0, 20])]
    bad = torch.zeros((2, 2, 64), dtype=torch.bool, device="cuda")
    bad[:, 0, 3] = bad[:, 0, 3 + 8] = bad[:, 1, 40] = True   # 3 and 11 are a pair; 40 is not rotated
    assert torch.equal(torch.isnan(b), bad)
    assert 20 in ops.select_pages(kv, c.q, c.seq_len, 3)[0, 0].tolist()
    assert torch.equal(ops.select_pages(kv, c.q, c.seq_len, 3).cpu(), ref.select(c, 3, 1, 1))
