"""The paged-cache operators against their formulas in 64 bits
(paged_reference.py, which also derives the tolerances)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import paged_reference as ref  # noqa: E402
from qweninferenceengine_b200 import QwenError, ops  # noqa: E402
from qweninferenceengine_b200._lib import QWEN_ERR_INVALID_ARGUMENT, QWEN_OK, lib  # noqa: E402

F16, BF16 = torch.float16, torch.bfloat16
DTYPES = [F16, BF16]


def status():
    return lib().qwen_ops_status(torch.cuda.current_stream().cuda_stream)


@pytest.fixture(autouse=True)
def clean_status(cuda):
    """No operator leaves a device-side report behind that its test did not read."""
    yield
    assert status() == QWEN_OK


# ------------------------------------------------------------------ append ---
def freqs(rot):
    return torch.tensor([1e6 ** (-2 * i / rot) for i in range(rot // 2)], dtype=torch.float32,
                        device="cuda")


def check_append(c, new, rot, interleaved, ragged, pad=0, strided=True, out=None):
    """Appends the last `new` positions of each sequence of a cache and checks every
    element of the pools, the bounds and q."""
    n, H, K, D, P = len(c.lens), c.heads, c.kv_heads, c.dim, c.page
    past = [x - y for x, y in zip(c.lens, new)]
    held, c.lens = c.lens, past
    c.make_bounds()
    c.lens = held
    rows = sum(new) + pad if ragged else n
    if strided:   # slices of one projection's rows
        qkv = c.randn(rows, (H + 2 * K) * D)
        q, k, v = (x.view(rows, -1, D) for x in qkv.split([H * D, K * D, K * D], dim=1))
    else:
        q, k, v = c.randn(rows, H, D), c.randn(rows, K, D), c.randn(rows, K, D)
    cu, row = None, []
    if ragged:
        cu = [0]
        for i in range(n):
            row += [(i, past[i] + j) for j in range(new[i])]
            cu.append(cu[-1] + new[i])
        cu = torch.tensor(cu, dtype=torch.int32, device="cuda")
    else:
        row = [(i, past[i]) if new[i] else None for i in range(n)]
    inv = freqs(rot)
    k0, v0, b0 = c.k.clone(), c.v.clone(), c.bounds.clone()
    q_in = q.clone()
    dst = torch.full((rows, H, D), 7.0, dtype=c.dtype, device="cuda") if out is None else q
    got = ops.rope_append_paged(c.handle(), q, k, v, c.seq_len, inv, cu_tokens=cu,
                                interleaved=interleaved, out=dst)
    assert got is dst
    live = [r for r, x in enumerate(row) if x is not None]
    pos = torch.tensor([row[r][1] for r in live], device="cuda")
    u = ref.U[c.dtype]
    yq, eq = ref.rotate(q_in[live], pos, inv, interleaved)
    yk, ek = ref.rotate(k[live], pos, inv, interleaved)
    off = (dst[live].double() - yq).abs() - (u * yq.abs() + 2 * eq + 1e-7)
    assert off.max().item() <= 0
    rest = [r for r in range(rows) if r not in set(live)]
    if rest and out is None:
        assert (dst[rest] == 7.0).all()
    for j, r in enumerate(live):
        i, p = row[r]
        page = int(c.table[i, p // P])
        k0[page, p % P] = c.k[page, p % P]          # checked here, with a tolerance
        off = (c.k[page, p % P].double() - yk[j]).abs() - (u * yk[j].abs() + 2 * ek[j] + 1e-7)
        assert off.max().item() <= 0
        v0[page, p % P] = v[r]
    same = lambda a, b: torch.equal(a.contiguous().view(torch.int16), b.contiguous().view(torch.int16))  # noqa: E731
    assert same(c.k, k0) and same(c.v, v0)
    for i in range(n):
        for j in range(past[i] // P, -(-c.lens[i] // P) if new[i] else 0):
            page = int(c.table[i, j])
            keys = c.k[page, : min(P, c.lens[i] - j * P)]
            b0[page, 0], b0[page, 1] = keys.amin(0), keys.amax(0)
    assert torch.equal(torch.nan_to_num(c.bounds.float(), 9e9), torch.nan_to_num(b0.float(), 9e9))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,K,D,P,rot,inter,hnd", [
    (12, 2, 128, 16, 128, False, False), (32, 8, 128, 64, 96, True, True),
    (14, 2, 64, 256, 64, False, True), (8, 8, 64, 32, 16, True, False), (16, 1, 128, 128, 64, False, False)])
def test_append_one_token(dtype, H, K, D, P, rot, inter, hnd):
    lens = [1, P, P + 1, 2 * P - 1, 0, 3 * P, 300]
    c = ref.Cache(1, lens, H, K, D, P, dtype, hnd)
    check_append(c, [min(x, 1) for x in lens], rot, inter, ragged=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,K,D,P,rot,inter,hnd", [
    (12, 2, 128, 16, 128, False, False), (12, 2, 128, 64, 128, False, True), (32, 8, 128, 256, 96, True, False),
    (14, 2, 64, 128, 64, False, True), (8, 8, 64, 32, 32, True, False)])
def test_append_ragged(dtype, H, K, D, P, rot, inter, hnd):
    lens = [1, P, P + 1, 2 * P - 1, 0, 3 * P, 300, 517, 64, 5]
    new = [1, P, 1, P, 0, 2 * P + 1, 300, 100, 0, 2]
    c = ref.Cache(2, lens, H, K, D, P, dtype, hnd)
    check_append(c, new, rot, inter, ragged=True, pad=5)


def test_append_one_long_prompt_and_dense_rows():
    c = ref.Cache(3, [2111], 12, 2, 128, 64, F16)
    check_append(c, [2100], 128, False, ragged=True, strided=False)


def test_append_in_place_and_far_positions():
    """q rotated in its own memory, at positions where an fp32 angle is off by 0.01."""
    c = ref.Cache(4, [200001, 131072], 12, 2, 128, 64, F16, spare=0)
    check_append(c, [70, 70], 128, False, ragged=True, strided=False, out="in place")


def test_append_a_page_begun_anew_forgets_its_bounds():
    c = ref.Cache(5, [17], 4, 2, 64, 16, BF16)
    c.make_bounds()
    c.bounds[int(c.table[0, 1])] = 1000.0     # what the page's last user left
    x = c.randn(1, 8, 64)
    ops.rope_append_paged(c.handle(), x[:, :4], x[:, 4:6], x[:, 6:], c.seq_len, freqs(64))
    page = int(c.table[0, 1])
    assert torch.equal(c.bounds[page, 0], c.k[page, 0]) and torch.equal(c.bounds[page, 1], c.k[page, 0])


def test_append_without_bounds_and_nothing_to_do():
    c = ref.Cache(6, [40, 3], 4, 2, 64, 16, F16)
    kv = c.handle()
    x = c.randn(43, 8, 64)
    cu = torch.tensor([0, 40, 43], dtype=torch.int32, device="cuda")
    ops.rope_append_paged(kv, x[:, :4], x[:, 4:6], x[:, 6:], c.seq_len, freqs(64), cu_tokens=cu)
    assert torch.equal(c.v[int(c.table[1, 0]), :3], x[40:, 6:])
    none = x[:0]
    cu.zero_()
    ops.rope_append_paged(kv, none[:, :4], none[:, 4:6], none[:, 6:], c.seq_len, freqs(64), cu_tokens=cu)


def test_append_reports_what_only_the_device_sees():
    c = ref.Cache(7, [20, 20, 20], 4, 2, 64, 16, F16)
    c.make_bounds()
    kv = c.handle()
    x = c.randn(3, 8, 64)
    out = torch.full((3, 4, 64), 7.0, dtype=F16, device="cuda")
    before = c.k.clone()
    c.seq_len[1] = 33                       # beyond two pages of 16
    ops.rope_append_paged(kv, x[:, :4], x[:, 4:6], x[:, 6:], c.seq_len, freqs(64), out=out)
    assert status() == QWEN_ERR_INVALID_ARGUMENT
    assert (out[1] == 7.0).all() and (out[0] != 7.0).any() and (out[2] != 7.0).any()
    c.seq_len[1] = 20
    for bad in (-1, c.n_pages, 2 ** 31 - 1):
        page = int(c.table[1, 1])
        c.table[1, 1] = bad
        c.k.copy_(before)
        ops.rope_append_paged(kv, x[:, :4], x[:, 4:6], x[:, 6:], c.seq_len, freqs(64), out=out)
        assert status() == QWEN_ERR_INVALID_ARGUMENT
        assert torch.equal(torch.nan_to_num(c.k[page]), torch.nan_to_num(before[page]))
        c.table[1, 1] = page
    for cu in ([0, 1, 9, 3], [0, 2, 1, 3], [-1, 1, 2, 3], [0, 3, 3, 3]):   # the last is in order: (3, 0, 0) new
        t = torch.tensor(cu, dtype=torch.int32, device="cuda")
        ops.rope_append_paged(kv, x[:, :4], x[:, 4:6], x[:, 6:], c.seq_len, freqs(64), cu_tokens=t, out=out)
        assert status() == (QWEN_OK if cu == [0, 3, 3, 3] else QWEN_ERR_INVALID_ARGUMENT)


# --------------------------------------------------------------- attention ---
LENS = [1, 15, 16, 17, 0, 127, 128, 129, 255, 256, 257, 511, 640, 1000, 2049]
HEADS = [(12, 2, 128), (32, 8, 128), (14, 2, 64), (8, 8, 64), (16, 1, 128), (34, 2, 128), (64, 1, 64), (9, 1, 64)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,K,D", HEADS)
@pytest.mark.parametrize("P,hnd", [(16, False), (64, True), (256, False)])
def test_attention_paged(dtype, H, K, D, P, hnd):
    c = ref.Cache(H * D + P, LENS, H, K, D, P, dtype, hnd)
    got = ops.attention_paged(c.handle(), c.q, c.seq_len, return_lse=True)
    ref.assert_attention(got, ref.attention(c, D ** -0.5))


@pytest.mark.parametrize("lens", [[1], [0], [70000], [5, 40001], [1] * 300, [0] * 9 + [33]])
@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_paged_shapes_of_batches(dtype, lens):
    c = ref.Cache(len(lens), lens, 12, 2, 128, 32, dtype)
    got = ops.attention_paged(c.handle(), c.q, c.seq_len, scale=0.2, return_lse=True)
    ref.assert_attention(got, ref.attention(c, 0.2))


def test_attention_paged_strided_rows_and_outputs():
    c = ref.Cache(11, [100, 1, 64], 12, 2, 128, 32, F16)
    wide = torch.full((3, 20, 128), 7.0, dtype=F16, device="cuda")
    wide[:, 4:16] = c.q
    out = torch.full((3, 14, 128), 7.0, dtype=F16, device="cuda")
    got = ops.attention_paged(c.handle(), wide[:, 4:16], c.seq_len, out=out[:, 1:13], return_lse=True)
    ref.assert_attention(got, ref.attention(c, 128 ** -0.5))
    assert (out[:, 0] == 7).all() and (out[:, 13] == 7).all()


def test_attention_paged_large_scores():
    """Scores of +-400: the running maximum moves far, most weights vanish."""
    c = ref.Cache(12, [700, 130], 12, 2, 128, 64, F16)
    c.q *= 4
    got = ops.attention_paged(c.handle(), c.q, c.seq_len, scale=1.0, return_lse=True)
    ref.assert_attention(got, ref.attention(c, 1.0))


def test_attention_paged_pool_beyond_32_bit_offsets():
    """Pages whose elements lie past 2^32: a pool of 2^33 bytes and more, two pages of it used."""
    n_pages = (1 << 32) // (256 * 2 * 128) + 40
    k = torch.empty((n_pages, 256, 2, 128), dtype=BF16, device="cuda")
    v = torch.empty_like(k)
    c = ref.Cache(13, [400], 12, 2, 128, 256, BF16)
    table = torch.tensor([[n_pages - 1, n_pages - 7]], dtype=torch.int32, device="cuda")
    for j in range(2):
        k[int(table[0, j])] = c.k[int(c.table[0, j])]
        v[int(table[0, j])] = c.v[int(c.table[0, j])]
    got = ops.attention_paged(ops.PagedKV(k, v, table), c.q, c.seq_len, return_lse=True)
    ref.assert_attention(got, ref.attention(c, 128 ** -0.5))


# ------------------------------------------------------------ shared prefix --
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,K,D,P,hnd", [(12, 2, 128, 16, False), (32, 8, 128, 64, True), (14, 2, 64, 256, False),
                                         (8, 8, 64, 32, True), (64, 1, 128, 128, False)])
@pytest.mark.parametrize("prefix", [0, 1, 100, 128, 1000])
def test_attention_prefix(dtype, H, K, D, P, hnd, prefix):
    lens = [0, 1, 17, 128, 300, 0, 5]
    c = ref.Cache(prefix + P, lens, H, K, D, P, dtype, hnd, prefix=prefix)
    got = ops.attention_prefix_paged(c.handle(), c.q, c.seq_len, c.prefix_pages, prefix, return_lse=True)
    ref.assert_attention(got, ref.attention(c, D ** -0.5))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,H,K,D,P,prefix", [(1, 12, 2, 128, 64, 5000), (22, 12, 2, 128, 64, 4097), (43, 12, 2, 128, 16, 777),
                                              (130, 16, 8, 64, 64, 1500), (300, 12, 2, 128, 128, 2100),
                                              (65, 64, 2, 128, 256, 3333)])
def test_attention_prefix_many_rows(dtype, n, H, K, D, P, prefix):
    lens = [(i * 37) % 90 for i in range(n)]
    c = ref.Cache(n, lens, H, K, D, P, dtype, prefix=prefix)
    got = ops.attention_prefix_paged(c.handle(), c.q, c.seq_len, c.prefix_pages, prefix, return_lse=True)
    ref.assert_attention(got, ref.attention(c, D ** -0.5))


def test_attention_prefix_large_and_tiny_scores():
    """Rows whose maximum lies in the prefix, in their own positions, or moves tile by tile."""
    c = ref.Cache(21, [300] * 40, 12, 2, 128, 64, F16, prefix=2000)
    c.q *= torch.linspace(0.01, 6, 40, device="cuda")[:, None, None].half()
    grow = torch.linspace(0.1, 3, 2000, device="cuda")
    for j in range(32):
        m = min(64, 2000 - 64 * j)
        c.k[int(c.prefix_pages[j]), :m] *= grow[64 * j: 64 * j + m, None, None].half()
    got = ops.attention_prefix_paged(c.handle(), c.q, c.seq_len, c.prefix_pages, 2000, scale=0.5, return_lse=True)
    ref.assert_attention(got, ref.attention(c, 0.5))


@pytest.mark.parametrize("scale", [-0.1, 0.0])
def test_attention_any_scale(scale):
    """A negative scale prefers the least products, a zero scale none."""
    c = ref.Cache(23, [100, 7, 0], 12, 2, 128, 32, BF16, prefix=300)
    kv = c.handle()
    got = ops.attention_prefix_paged(kv, c.q, c.seq_len, c.prefix_pages, 300, scale=scale, return_lse=True)
    ref.assert_attention(got, ref.attention(c, scale))
    c.prefix = 0
    got = ops.attention_paged(kv, c.q, c.seq_len, scale=scale, return_lse=True)
    ref.assert_attention(got, ref.attention(c, scale))


def test_attention_prefix_is_paged_attention_of_the_whole():
    """The same positions through one table: prefix pages, then a sequence's own."""
    c = ref.Cache(22, [50, 64, 1, 0], 12, 2, 128, 64, BF16, prefix=640)
    got = ops.attention_prefix_paged(c.handle(), c.q, c.seq_len, c.prefix_pages, 640)
    table = torch.cat((c.prefix_pages[None].expand(4, -1), c.table), dim=1).contiguous()
    whole = ops.attention_paged(ops.PagedKV(c.k, c.v, table), c.q, c.seq_len + 640)
    assert (got.double() - whole.double()).abs().max().item() <= 4 * ref.U[BF16] * whole.abs().max().item()


def test_one_table_for_appending_and_for_the_prefix():
    """Rows that begin with the prefix's pages: new tokens are rotated at their positions in
    the whole, and the prefix call reads the columns behind."""
    n_prefix, P = 5, 32
    c = ref.Cache(23, [50, 64, 1, 200], 12, 2, 128, P, F16, prefix=n_prefix * P)
    table = torch.cat((c.prefix_pages[None].expand(4, -1), c.table), dim=1).contiguous()
    x, whole, inv = c.randn(4, 16, 128), c.seq_len + n_prefix * P, freqs(128)
    c.q = ops.rope_append_paged(ops.PagedKV(c.k, c.v, table), x[:, :12], x[:, 12:14], x[:, 14:], whole, inv)
    yq, eq = ref.rotate(x[:, :12], whole.double() - 1, inv, False)
    assert ((c.q.double() - yq).abs() - (ref.U[F16] * yq.abs() + 2 * eq + 1e-7)).max().item() <= 0
    own = ops.PagedKV(c.k, c.v, table[:, n_prefix:])
    got = ops.attention_prefix_paged(own, c.q, c.seq_len, table[0, :n_prefix], n_prefix * P, return_lse=True)
    ref.assert_attention(got, ref.attention(c, 128 ** -0.5))


def test_prefix_beside_many_own_positions():
    """Own positions for which the SMs left beside the prefix are too few, and enough."""
    for lens, prefix in (([2000] * 60, 3000), ([20] * 200, 9000), ([3000] + [0] * 199, 9000), ([64] * 3, 100000)):
        c = ref.Cache(24, lens, 12, 2, 128, 128, BF16, prefix=prefix)
        got = ops.attention_prefix_paged(c.handle(), c.q, c.seq_len, c.prefix_pages, prefix, return_lse=True)
        ref.assert_attention(got, ref.attention(c, 128 ** -0.5))


# ----------------------------------------------------------- page selection --
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,K,D", [(12, 2, 128), (32, 8, 128), (14, 2, 64), (8, 8, 64), (16, 1, 128), (64, 1, 64)])
@pytest.mark.parametrize("P,S,first,last", [(16, 7, 1, 1), (64, 4, 0, 0), (16, 3, 1, 2), (32, 40, 2, 5), (16, 1, 0, 0)])
def test_select_and_sparse(dtype, H, K, D, P, S, first, last):
    lens = [1, 16, 17, 0, 129, 640, 1000, 2500]
    c = ref.Cache(H + P + S, lens, H, K, D, P, dtype, hnd=P == 32)
    c.make_bounds()
    kv = c.handle()
    pages = ops.select_pages(kv, c.q, c.seq_len, S, n_first=first, n_last=last)
    assert torch.equal(pages.cpu(), ref.select(c, S, first, last))
    got = ops.attention_sparse_paged(kv, c.q, c.seq_len, pages, return_lse=True)
    ref.assert_attention(got, ref.attention(c, D ** -0.5, lists=pages))


@pytest.mark.parametrize("length", [16 * 300, 16 * 1025 - 3, 16 * 4000, 16 * 8192])
@pytest.mark.parametrize("S", [2, 33, 256, 1000])
def test_select_long(length, S):
    c = ref.Cache(length + S, [length, 16 * 50, length // 2], 12, 2, 64, 16, BF16)
    c.make_bounds()
    assert torch.equal(ops.select_pages(c.handle(), c.q, c.seq_len, S).cpu(), ref.select(c, S, 1, 1))


@pytest.mark.parametrize("levels", [1, 2, 7])
def test_select_ties_go_to_the_lower_page(levels):
    c = ref.Cache(31, [16 * 900], 4, 2, 64, 16, F16)
    c.make_bounds()
    # bounds of few kinds: whole runs of pages with the very same score
    kinds = c.randn(levels, 2, 2, 64)
    kinds = torch.stack((kinds.amin(1), kinds.amax(1)), dim=1)
    pick = torch.randint(0, levels, (900,), generator=c.g, device="cuda")
    c.bounds[c.table[0].long()] = kinds[pick]
    for S in (3, 64, 500, 899):
        assert torch.equal(ops.select_pages(c.handle(), c.q, c.seq_len, S).cpu(), ref.select(c, S, 1, 1))


def test_select_extreme_scores():
    """Infinite and NaN bounds, equal extremes, a score range of 2^30."""
    c = ref.Cache(32, [16 * 400], 4, 2, 64, 16, F16)
    c.make_bounds()
    b = c.bounds
    t = c.table[0].long()
    b[t[5]] *= 1000
    b[t[7], 1] = math.inf
    b[t[9], 0] = -math.inf
    b[t[11]] = math.nan
    b[t[100:200]] *= 2.0 ** -14
    b[t[200:220]] = 0
    c.q[0, 1] = 0
    c.q += 2.0 ** -20
    for S in (4, 30, 150, 260, 399):
        assert torch.equal(ops.select_pages(c.handle(), c.q, c.seq_len, S).cpu(), ref.select(c, S, 1, 1))


def test_sparse_lists_of_any_form():
    """Holes, any order, a column listed twice, columns past the end, empty lists."""
    c = ref.Cache(33, [500, 100, 300, 0], 12, 2, 128, 32, F16)
    pages = torch.tensor([[[3, -1, 0, 15, -1, 2], [15, 14, 13, 1, 0, 7]],
                          [[-1] * 6, [3, -1, -1, -1, -1, 0]],
                          [[9, 8, -1, -1, 12, 15], [4, 4, 2, 4, -1, 10]],
                          [[0, 1, 2, 3, 4, 5], [-1] * 6]], dtype=torch.int32, device="cuda")
    got = ops.attention_sparse_paged(c.handle(), c.q, c.seq_len, pages, return_lse=True)
    ref.assert_attention(got, ref.attention(c, 128 ** -0.5, lists=pages))


def test_nan_keys_show_in_their_rows_alone():
    """A NaN among the positions that count gives NaN for the heads that read it, also
    where it is all a sequence or a prefix has."""
    for prefix in (0, 1, 130):
        c = ref.Cache(34, [1, 400, 0, 33], 12, 2, 128, 32, F16, prefix=prefix)
        kv = c.handle()
        c.k[int(c.table[0, 0]), 0, 1] = math.nan
        c.k[int(c.table[1, 7]), 3, 0] = math.nan
        bad = torch.zeros((4, 12), dtype=torch.bool, device="cuda")
        bad[0, 6:] = bad[1, :6] = True
        for shared in (False, True):
            if shared and prefix:
                c.k[int(c.prefix_pages[0]), 0, 1] = math.nan
                bad[:, 6:] = True
            out, lse = ops.attention_prefix_paged(kv, c.q, c.seq_len, c.prefix_pages, prefix, return_lse=True)
            assert torch.isnan(out[bad]).all() and torch.isnan(lse[bad]).all()
            want, want_lse, tol, lse_tol = ref.attention(c, 128 ** -0.5)
            ref.assert_attention((out[~bad], lse[~bad]), (want[~bad], want_lse[~bad], tol[~bad], lse_tol[~bad]))


def test_attention_in_place():
    c = ref.Cache(35, [5000, 1, 0, 300], 12, 2, 128, 32, BF16, prefix=500)
    kv, q = c.handle(), c.q.clone()
    c.prefix, want = 0, {}
    want[0] = ref.attention(c, 128 ** -0.5)
    c.prefix = 500
    want[500] = ref.attention(c, 128 ** -0.5)
    for prefix in (0, 500):
        x = q.clone()
        got = ops.attention_prefix_paged(kv, x, c.seq_len, c.prefix_pages, prefix, out=x, return_lse=True)
        assert got[0] is x
        ref.assert_attention(got, want[prefix])


# ------------------------------------------------- reports, streams, graphs --
def test_attention_reports_what_only_the_device_sees():
    c = ref.Cache(41, [40, 60, 33], 12, 2, 128, 16, F16, width=4)
    c.make_bounds()
    kv = c.handle()
    whole = ref.attention(c, 128 ** -0.5)
    calls = [lambda o: ops.attention_paged(kv, c.q, c.seq_len, out=o),
             lambda o: ops.attention_prefix_paged(kv, c.q, c.seq_len, c.table[0, :1].contiguous(), 3, out=o),
             lambda o: ops.attention_sparse_paged(kv, c.q, c.seq_len, columns, out=o)]
    columns = torch.arange(4, dtype=torch.int32, device="cuda").expand(3, 2, 4).contiguous()
    for call in calls:
        out = torch.full((3, 12, 128), 7.0, dtype=F16, device="cuda")
        for bad in (65, -1, 2 ** 31 - 1):
            c.seq_len[1] = bad
            call(out)
            assert status() == QWEN_ERR_INVALID_ARGUMENT
            assert (out[1] == 7).all() and (out[0] != 7).any() and (out[2] != 7).any()
        c.seq_len[1] = 60
        call(out)
        assert status() == QWEN_OK
    # a page outside the pool: reported, its positions left out, the others' rows right
    page = int(c.table[1, 3])
    for bad in (-1, c.n_pages, 2 ** 31 - 1):
        c.table[1, 3] = bad
        out, lse = ops.attention_paged(kv, c.q, c.seq_len, return_lse=True)
        assert status() == QWEN_ERR_INVALID_ARGUMENT
        left = ref.Cache(41, [40, 60, 33], 12, 2, 128, 16, F16, width=4)
        left.lens = [40, 48, 33]
        ref.assert_attention((out, lse), ref.attention(left, 128 ** -0.5))
        ops.select_pages(kv, c.q, c.seq_len, 3)
        assert status() == QWEN_ERR_INVALID_ARGUMENT
    c.table[1, 3] = page
    columns[2, 1, 0] = 4
    ops.attention_sparse_paged(kv, c.q, c.seq_len, columns)
    assert status() == QWEN_ERR_INVALID_ARGUMENT
    # ... in a shared prefix, for every row
    shared = ref.Cache(42, [40, 0, 33], 12, 2, 128, 16, F16, prefix=300)
    pages = shared.prefix_pages.clone()
    pages[3], pages[18] = c.n_pages + 100, -1
    got = ops.attention_prefix_paged(shared.handle(), shared.q, shared.seq_len, pages, 300, return_lse=True)
    assert status() == QWEN_ERR_INVALID_ARGUMENT
    keep = [i for i in range(19) if i not in (3, 18)]
    shared.prefix_pages, shared.prefix = shared.prefix_pages[keep], 17 * 16
    ref.assert_attention(got, ref.attention(shared, 128 ** -0.5))
    ref.assert_attention(ops.attention_paged(kv, c.q, c.seq_len, return_lse=True), whole)


def one_step(c, kv, qkv, inv, S=6):
    """A decode step's chain over one layer: append, dense, sparse and shared-prefix reads."""
    q = ops.rope_append_paged(kv, qkv[:, :12], qkv[:, 12:14], qkv[:, 14:], c.seq_len, inv)
    pages = ops.select_pages(kv, q, c.seq_len, S)
    sparse = ops.attention_sparse_paged(kv, q, c.seq_len, pages, return_lse=True)
    dense = ops.attention_paged(kv, q, c.seq_len, return_lse=True)
    prefix = ops.attention_prefix_paged(kv, q, c.seq_len, c.prefix_pages, c.prefix, return_lse=True)
    return q, pages, sparse, dense, prefix


def check_step(c, got, S=6):
    q, pages, sparse, dense, prefix = got
    c.q, c.lens = q, c.seq_len.tolist()
    n_prefix, c.prefix = c.prefix, 0
    assert torch.equal(pages.cpu(), ref.select(c, S, 1, 1))
    ref.assert_attention(sparse, ref.attention(c, 128 ** -0.5, lists=pages))
    ref.assert_attention(dense, ref.attention(c, 128 ** -0.5))
    c.prefix = n_prefix
    ref.assert_attention(prefix, ref.attention(c, 128 ** -0.5))


def serving_cache(seed, dtype):
    c = ref.Cache(seed, [300, 47, 16, 129], 12, 2, 128, 16, dtype, prefix=333, width=40)
    c.make_bounds()
    return c


@pytest.mark.parametrize("dtype", DTYPES)
def test_operators_together(dtype):
    """Prompts appended, then decode steps: each reads what the ones before wrote."""
    c = ref.Cache(51, [0, 0, 0, 0], 12, 2, 128, 16, dtype, prefix=333, width=40)
    c.make_bounds()
    kv, inv = c.handle(), freqs(128)
    lens = [300, 47, 16, 129]
    x = c.randn(sum(lens), 16, 128)
    c.seq_len.copy_(torch.tensor(lens))
    cu = torch.tensor([0, 300, 347, 363, 492], dtype=torch.int32, device="cuda")
    ops.rope_append_paged(kv, x[:, :12], x[:, 12:14], x[:, 14:], c.seq_len, inv, cu_tokens=cu)
    for _ in range(3):
        c.seq_len += 1
        got = one_step(c, kv, c.randn(4, 16, 128), inv)
        check_step(c, got)


def test_captured_and_replayed():
    """Two graphs over one memory pool, captured once, replayed over growing lengths."""
    inv = freqs(128)
    caches, graphs, outs, ins = [], [], [], []
    pool = torch.cuda.graph_pool_handle()
    for seed in (61, 62):
        c = serving_cache(seed, F16)
        qkv = c.randn(4, 16, 128)
        kv = c.handle()
        c.seq_len += 1
        one_step(c, kv, qkv, inv)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            outs.append(one_step(c, kv, qkv, inv))
        caches.append((c, kv))
        graphs.append(g)
        ins.append(qkv)
    for step in range(3):
        for (c, kv), g, qkv, out in zip(caches, graphs, ins, outs):
            c.seq_len += 1
            qkv.copy_(c.randn(4, 16, 128))
            g.replay()
            check_step(c, out)


@pytest.mark.parametrize("fill", [0, 0xFF, None])
def test_workspace_of_any_contents(fill, monkeypatch):
    """One workspace for all calls, whatever it holds; then shared by two captured graphs."""
    sized = ops._workspace
    memory = torch.randint(0, 256, (1 << 26,), dtype=torch.uint8, device="cuda")
    if fill is not None:
        memory.fill_(fill)

    def given(kv, query, *sizes):
        need = sized(kv, query, *sizes)[1]
        assert need <= memory.numel()
        return memory, need

    monkeypatch.setattr(ops, "_workspace", given)
    inv = freqs(128)
    work = []
    for seed in (63, 64):
        c = serving_cache(seed, BF16)
        c.seq_len += 1
        kv, qkv = c.handle(), c.randn(4, 16, 128)
        check_step(c, one_step(c, kv, qkv, inv))
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = one_step(c, kv, qkv, inv)
        work.append((c, g, out, qkv))   # the graph reads qkv's memory
    for _ in range(3):
        for c, g, out, _ in work:
            g.replay()
            check_step(c, out)


def test_two_streams_at_once():
    """The same operators on two streams with nothing between them, again and again."""
    inv = freqs(128)
    work = []
    for seed in (71, 72):
        c = serving_cache(seed, BF16)
        c.seq_len += 1
        work.append((c, c.handle(), c.randn(4, 16, 128), torch.cuda.Stream()))
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(20):
        for i, (c, kv, qkv, st) in enumerate(work):
            with torch.cuda.stream(st):
                got[i] = one_step(c, kv, qkv, inv)
    torch.cuda.synchronize()
    for (c, *_), g in zip(work, got):
        check_step(c, g)


def test_same_call_same_bits():
    c = ref.Cache(81, [3000, 17, 900, 1], 12, 2, 128, 64, F16, prefix=5000)
    kv = c.handle()
    for call in (lambda: ops.attention_paged(kv, c.q, c.seq_len),
                 lambda: ops.attention_prefix_paged(kv, c.q, c.seq_len, c.prefix_pages, 5000)):
        first = call()
        for _ in range(5):
            assert torch.equal(call(), first)


def test_profiling_command_runs_them(capsys):
    from qweninferenceengine_b200.profiling import run_paged

    run_paged(batch=3, ctx=100, page=16, prefix=300, select=4, reps=2)
    out = capsys.readouterr().out
    for name in ("rope_append_paged", "attention_paged", "attention_prefix_paged", "select_pages",
                 "attention_sparse_paged"):
        assert name in out


# ------------------------------------------------------------------ refusals --
def test_python_refusals():
    c = ref.Cache(91, [40, 20], 12, 2, 128, 16, F16, prefix=20)
    c.make_bounds()
    kv = c.handle()
    inv = freqs(128)
    x = c.randn(2, 16, 128)
    bad_value = [
        lambda: ops.PagedKV(c.k, c.v[:, :, :1], c.table),
        lambda: ops.PagedKV(c.k, c.v.transpose(0, 1).contiguous().transpose(0, 1), c.table),
        lambda: ops.PagedKV(c.k.float(), c.v.float(), c.table),
        lambda: ops.PagedKV(c.k, c.v.to(BF16), c.table),
        lambda: ops.PagedKV(c.k, c.v, c.table.long()),
        lambda: ops.PagedKV(c.k, c.v, c.table.T),
        lambda: ops.PagedKV(c.k, c.v, c.table.cpu()),
        lambda: ops.PagedKV(c.k, c.v, c.table, c.bounds[:-1]),
        lambda: ops.PagedKV(c.k, c.v, c.table, c.bounds.float()),
        lambda: ops.PagedKV(c.k.transpose(2, 3), c.v.transpose(2, 3), c.table),
        lambda: ops.attention_paged(kv, c.q.to(BF16), c.seq_len),
        lambda: ops.attention_paged(kv, c.q[:1], c.seq_len),
        lambda: ops.attention_paged(kv, c.q[..., :64], c.seq_len),
        lambda: ops.attention_paged(kv, c.q.transpose(0, 1).contiguous().transpose(0, 1), c.seq_len),
        lambda: ops.attention_paged(kv, c.q, c.seq_len[:1]),
        lambda: ops.attention_paged(kv, c.q, c.seq_len.long()),
        lambda: ops.attention_paged(kv, c.q, c.seq_len.cpu()),
        lambda: ops.attention_paged(kv, c.q, c.seq_len, out=torch.empty_like(c.q).float()),
        lambda: ops.attention_prefix_paged(kv, c.q, c.seq_len, c.prefix_pages, 33),
        lambda: ops.attention_prefix_paged(kv, c.q, c.seq_len, c.prefix_pages, -1),
        lambda: ops.attention_prefix_paged(kv, c.q, c.seq_len, c.prefix_pages.long(), 20),
        lambda: ops.select_pages(kv, c.q, c.seq_len, 0),
        lambda: ops.select_pages(kv, c.q, c.seq_len, 4, n_first=-1),
        lambda: ops.select_pages(kv, c.q, c.seq_len, 4, out=torch.empty((2, 2, 3), dtype=torch.int32, device="cuda")),
        lambda: ops.attention_sparse_paged(kv, c.q, c.seq_len, torch.zeros((2, 1, 4), dtype=torch.int32, device="cuda")),
        lambda: ops.attention_sparse_paged(kv, c.q, c.seq_len, torch.zeros((2, 2, 4), dtype=torch.int64, device="cuda")),
        lambda: ops.rope_append_paged(kv, x[:, :12], x[:1, 12:14], x[:, 14:], c.seq_len, inv),
        lambda: ops.rope_append_paged(kv, x[:, :12], x[:, 12:13], x[:, 14:], c.seq_len, inv),
        lambda: ops.rope_append_paged(kv, x[:, :12], x[:, 12:14], x[:, 14:], c.seq_len, inv.double()),
        lambda: ops.rope_append_paged(kv, x[:, :12], x[:, 12:14], x[:, 14:], c.seq_len, inv, cu_tokens=c.seq_len),
        lambda: ops.rope_append_paged(kv, x[:, :12], x[:, 12:14], x[:, 14:], c.seq_len, inv, out=x[:, :11]),
    ]
    for call in bad_value:
        with pytest.raises(ValueError):
            call()
    bad_status = [
        lambda: ops.attention_paged(kv, c.randn(2, 13, 128), c.seq_len),
        lambda: ops.attention_paged(kv, c.randn(2, 130, 128), c.seq_len),
        lambda: ops.attention_sparse_paged(kv, c.q, c.seq_len, torch.zeros((2, 2, 0), dtype=torch.int32, device="cuda")),
        lambda: ops.select_pages(kv, c.q, c.seq_len, 3, n_first=2, n_last=2),
        lambda: ops.select_pages(ops.PagedKV(c.k, c.v, c.table), c.q, c.seq_len, 3),
        lambda: ops.rope_append_paged(kv, x[:, :12], x[:, 12:14], x[:, 14:], c.seq_len, freqs(24)),
        lambda: ops.rope_append_paged(kv, x[:, :12], x[:, 12:14], x[:, 14:], c.seq_len, freqs(144)),
        lambda: ops.rope_append_paged(kv, x[:1, :12], x[:1, 12:14], x[:1, 14:], c.seq_len, inv),
    ]
    for call in bad_status:
        with pytest.raises(QwenError) as e:
            call()
        assert e.value.code == QWEN_ERR_INVALID_ARGUMENT
