"""Calls of the 4-bit cache's operators at the sizes where work is divided another way, and
such as the documents allow and nothing else tests."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

import paged_q4_reference as ref  # noqa: E402
from qweninferenceengine_b200 import ops  # noqa: E402
from qweninferenceengine_b200._lib import QWEN_OK, lib  # noqa: E402
from test_gpu_paged_q4 import check_append, check_evict, freqs, ints  # noqa: E402

F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(autouse=True)
def clean_status(cuda):
    yield
    assert lib().qwen_ops_status(torch.cuda.current_stream().cuda_stream) == QWEN_OK


def test_a_batch_that_ran_empty():
    c = ref.Cache(1, [20], 12, 2, 128, 16, F16, kept=True)
    kv = ops.PagedKVQ4(c.pool, c.table[:0], F16, c.weights[:0], c.positions[:0])
    lens, x = c.seq_len[:0], c.randn(1, 16, 128)[:0]
    before = c.pool.clone()
    for positions in (None, ints(), torch.zeros((1, 0), dtype=torch.int32, device="cuda")):
        q = ops.rope_append_paged_q4(kv, x[:, :12], x[:, 12:14], x[:, 14:], lens, freqs(128), positions=positions)
        assert q.shape == (0, 12, 128)
    out, lse = ops.attention_paged_q4(kv, c.q[:0], lens, return_lse=True)
    assert out.shape == (0, 12, 128) and lse.shape == (0, 12)
    assert ops.evict_paged_q4(kv, lens, 5).shape == (0,)
    k, v = ops.expand_paged_q4(kv, lens)
    assert k.shape == v.shape == (0, 2, 128)
    assert torch.equal(c.pool, before)


def test_as_many_sequences_as_a_call_takes():
    """65535 sequences of one page, in the order of the pool."""
    n, H, D, P = 65535, 2, 64, 16
    g = torch.Generator(device="cuda").manual_seed(3)
    lens = torch.randint(0, P + 1, (n,), generator=g, device="cuda").to(torch.int32)
    lens[0], lens[-1] = P, P
    pool = torch.zeros((n, 1, 1, 20 * D), dtype=torch.uint8, device="cuda")
    table = torch.arange(n, dtype=torch.int32, device="cuda").view(n, 1)
    weights = torch.rand((n, 1, P), generator=g, device="cuda")
    positions = torch.zeros((n, 1, P), dtype=torch.int32, device="cuda")
    kv = ops.PagedKVQ4(pool, table, F16, weights, positions)
    cu = torch.cat((torch.zeros(1, dtype=torch.int64, device="cuda"), lens.cumsum(0))).to(torch.int32)
    rows = int(cu[-1])
    x = torch.randn((rows, H + 2, D), generator=g, device="cuda").half()
    ops.rope_append_paged_q4(kv, x[:, :H], x[:, H: H + 1], x[:, H + 1:], lens, torch.zeros(32, device="cuda"), cu_tokens=cu)
    k, v = ops.expand_paged_q4(kv, lens, cu, n_rows=rows)
    for got, want in ((k, x[:, H: H + 1]), (v, x[:, H + 1:])):
        code, step, low = ref.quantise(want)
        value = low.double()[..., None] + code.double() * step.double()[..., None]
        assert torch.equal(got, ref.to_type(value.flatten(-2), F16))
    at = torch.arange(P, device="cuda")
    there = at < lens[:, None]
    assert (weights[:, 0][there] == 0).all() and torch.equal(positions[:, 0][there], at.expand(n, P)[there].int())
    q = torch.randn((n, H, D), generator=g, device="cuda").half()
    before = weights.clone()
    out, lse = ops.attention_paged_q4(kv, q, lens, return_lse=True)
    kk, vv = (torch.zeros((n, P, D), dtype=torch.float64, device="cuda") for _ in range(2))
    kk[there], vv[there] = k[:, 0].double(), v[:, 0].double()
    s = (q.double() @ kk.transpose(1, 2) * D ** -0.5).masked_fill(~there[:, None], -torch.inf)
    w = torch.softmax(s, -1).nan_to_num(0.0)
    # (k and v as expanded are off by half a step of fp16 each, 2^-11: of values up to 5 and scores up to 10)
    assert (out.double() - w @ vv).abs().max().item() < 0.03
    assert ((lse.double() - torch.logsumexp(s, -1)).nan_to_num(0.0, 0.0, 0.0)).abs().max().item() < 0.03
    assert torch.equal(torch.isneginf(lse), (lens == 0)[:, None].expand(n, H))
    assert ((weights - before)[:, 0].double() - w.sum(1)).abs().max().item() < 0.03
    new = ops.evict_paged_q4(kv, lens, 7, 1, 2)
    assert torch.equal(new, lens.clamp(max=7))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lens,H,K,D,P", [
    ([128 * 444], 8, 1, 64, 256), ([128 * 443 + 1], 6, 1, 128, 16), ([127, 129] * 160, 4, 2, 64, 32),
    ([1] * 500, 7, 1, 128, 16), ([128] * 444, 3, 1, 64, 64), ([128 * 148, 5, 128 * 30 + 7], 12, 2, 128, 128),
    ([40] * 1300, 2, 2, 64, 16)])
def test_attention_where_its_division_changes(dtype, lens, H, K, D, P):
    c = ref.Cache(4, lens, H, K, D, P, dtype, kept=True)
    before = c.weights.clone()
    got = ops.attention_paged_q4(c.handle(), c.q, c.seq_len, return_lse=True)
    r = ref.attention(c, D ** -0.5)
    ref.check_attention(got, r)
    ref.check_weights(c.weights, before, r)


def test_more_sequences_than_lanes_search():
    """Over 256 sequences rows find theirs by halving; many have nothing new."""
    lens = [(7 * i) % 23 for i in range(400)]
    new = [min(x, (3 * i) % 5) for i, x in enumerate(lens)]
    c = ref.Cache(5, lens, 4, 1, 64, 16, BF16, kept=True)
    check_append(c, new, 64, False, ragged=True, axes=2, far=300, pad=3)
    cu = [0]
    for x in lens:
        cu.append(cu[-1] + x)
    k, v = ops.expand_paged_q4(c.handle(), c.seq_len, ints(*cu), n_rows=cu[-1])
    for i in (0, 1, 257, 399):
        want = c.rows(i, c.all_slots(i))
        assert torch.equal(k[cu[i]: cu[i + 1]], ref.to_type(want[0], BF16))
        assert torch.equal(v[cu[i]: cu[i + 1]], ref.to_type(want[1], BF16))


def test_expand_of_more_rows_than_are_looked_up_at_once():
    c = ref.Cache(6, [90000, 3], 2, 1, 64, 256, F16)
    k, v = ops.expand_paged_q4(c.handle(), c.seq_len, ints(0, 90000, 90003), n_rows=90003)
    for i, at in ((0, 0), (1, 90000)):
        want = c.rows(i, c.all_slots(i))
        assert torch.equal(k[at: at + c.lens[i]], ref.to_type(want[0], F16))
        assert torch.equal(v[at: at + c.lens[i]], ref.to_type(want[1], F16))


def test_tables_and_pools_of_other_strides():
    """A table that is part of a wider one, a pool that holds three layers' pages side by
    side, one row of positions for all axes, a single axis as a matrix."""
    c = ref.Cache(7, [70, 33], 4, 2, 64, 16, F16, kept=True)
    wide = torch.full((2, c.width + 5), -7, dtype=torch.int32, device="cuda")
    wide[:, 2: 2 + c.width] = c.table
    c.table = wide[:, 2: 2 + c.width]
    layers = torch.full((c.n_pages, 3, 2, 1, 1280), 255, dtype=torch.uint8, device="cuda")
    layers[:, 1] = c.pool
    c.pool = layers[:, 1]
    want = ref.attention(c, 0.125)
    before = c.weights.clone()
    ref.check_attention(ops.attention_paged_q4(c.handle(), c.q, c.seq_len, return_lse=True), want)
    ref.check_weights(c.weights, before, want)
    x = c.randn(2, 8, 64)
    same = c.randn(2, 8, 64)
    same.copy_(x)
    pos = ints(500, 900)
    which = (torch.arange(32, device="cuda") % 3).to(torch.uint8)
    outs = []
    for p, w in ((pos, None), (pos[None], None), (pos.expand(3, 2), which), (pos.repeat(3, 1), which)):
        outs.append(ops.rope_append_paged_q4(c.handle(), x[:, :4], x[:, 4:6], x[:, 6:], c.seq_len, freqs(64),
                                             positions=p, pair_axis=w))
        outs.append(c.pool.clone())
    for i in range(2, 8):
        assert torch.equal(outs[i], outs[i % 2])
    assert torch.equal(x, same) and (layers[:, 0] == 255).all() and (layers[:, 2] == 255).all()


@pytest.mark.parametrize("kept", [False, True])
def test_workspaces_of_any_contents(kept):
    c = ref.Cache(8, [5000, 0, 300, 128 * 20], 16, 2, 64, 64, F16, kept=kept)
    kv = c.handle()
    need = lib().qwen_attention_paged_q4_workspace(kv.ref, 16)
    evict = lib().qwen_evict_paged_q4_workspace(kv.ref, 100)
    want, lse = ref.attention(c, 0.125), torch.empty(4, 16, device="cuda")
    out = torch.empty(4, 16, 64, dtype=F16, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    ws = torch.empty(max(need, evict), dtype=torch.uint8, device="cuda")
    for fill in (0, 255, 1, "random"):
        if fill == "random":
            ws.copy_(torch.randint(0, 256, ws.shape, generator=c.g, device="cuda").to(torch.uint8))
        else:
            ws.fill_(fill)
        before = c.weights.clone() if kept else None
        assert lib().qwen_attention_paged_q4(kv.ref, c.q.data_ptr(), 1024, out.data_ptr(), 1024, lse.data_ptr(), 16,
                                             c.seq_len.data_ptr(), 0.125, ws.data_ptr(), need, st) == QWEN_OK
        ref.check_attention((out, lse), want)
        if kept:
            ref.check_weights(c.weights, before, want)


def test_weights_grow_with_each_replay():
    c = ref.Cache(9, [300, 77], 12, 2, 128, 64, BF16, kept=True)
    kv, want, before = c.handle(), ref.attention(c, 128 ** -0.5), c.weights.clone()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        out = ops.attention_paged_q4(kv, c.q, c.seq_len)
    stream.synchronize()
    c.weights.copy_(before)
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]   # two with a workspace each
    for graph in graphs:
        with torch.cuda.graph(graph, stream=stream):
            out = ops.attention_paged_q4(kv, c.q, c.seq_len)
    for i in range(6):
        graphs[i % 2].replay()
        if i == 3:
            ops.attention_paged_q4(kv, c.q, c.seq_len)
    torch.cuda.synchronize()
    ref.check_attention((out, None), want)
    off = (c.weights.double() - before.double() - 7 * want[2]).abs() - 7 * want[5] - 2.0 ** -20 * (before + 7 * want[2])
    assert off.max().item() <= 0


@pytest.mark.parametrize("lens,width,keep", [
    ([33], 2500, 32), ([40000], 2500, 8), ([4097, 4095], 300, 4096), ([31, 64, 65], 2500, 64),
    ([16384 * 4 + 5], 4200, 3000), ([600] * 40, 64, 599), ([16385] * 30, 1100, 5), ([200], 13, 4000)])
def test_evict_where_its_division_changes(lens, width, keep):
    """Rows over several CTAs, some without slots, rows beyond what shared memory holds,
    budgets beyond the cache."""
    c = ref.Cache(10, lens, 2, 1, 64, 16, F16, width=width, kept=True)
    for i, x in enumerate(lens):
        c.positions[i, :, :x] = torch.randperm(x, generator=c.g, device="cuda").to(torch.int32)
    check_evict(c, keep, 3, keep // 3)


def test_evict_ties_across_the_ctas_of_a_row():
    c = ref.Cache(11, [50000], 2, 1, 64, 256, BF16, kept=True)
    c.weights.copy_(torch.randint(0, 2, c.weights.shape, generator=c.g, device="cuda").float())
    check_evict(c, 40000, 0, 0)
    c.weights.fill_(1.0)
    check_evict(c, 20000, 0, 10)
    c.positions.fill_(7)     # all guarded
    c.weights.copy_(torch.randint(0, 3, c.weights.shape, generator=c.g, device="cuda").float())
    check_evict(c, 30000, 0, 1)


def test_another_stream_than_the_current_devices_first():
    c = ref.Cache(12, [700, 64], 12, 2, 128, 64, F16, kept=True)
    want, before = ref.attention(c, 128 ** -0.5), c.weights.clone()
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        got = ops.attention_paged_q4(c.handle(), c.q, c.seq_len, return_lse=True)
        new = ops.evict_paged_q4(c.handle(), c.seq_len, 64, 1, 8)
        rows = ops.expand_paged_q4(c.handle(), new, ints(0, 64, 128), n_rows=128)
        torch.cuda.current_stream().synchronize()
    ref.check_attention(got, want)
    assert new.tolist() == [64, 64]
    c.lens = [64, 64]
    for i in range(2):
        assert torch.equal(rows[0][64 * i: 64 * i + 64], ref.to_type(c.rows(i, c.all_slots(i))[0], F16))
    assert torch.isfinite(before).all()


def test_the_library_reads_a_plain_structure():
    """qwen_paged_kv_q4 as C lays it out is what the wrapper packs."""
    from qweninferenceengine_b200._lib import PagedKVQ4Struct

    c = ref.Cache(13, [20], 4, 2, 64, 32, BF16, kept=True, head_gap=1)
    s = PagedKVQ4Struct.from_buffer_copy(c.handle().ref)
    assert ctypes.sizeof(PagedKVQ4Struct) == 80 == len(c.handle().ref)
    assert (s.pool, s.weights, s.positions, s.page_table) == tuple(
        x.data_ptr() for x in (c.pool, c.weights, c.positions, c.table))
    assert (s.page_stride, s.head_stride) == (3 * 2 * 1280, 2 * 1280)
    assert (s.n_pages, s.page_size, s.n_kv_heads, s.head_dim, s.n_seq, s.max_pages, s.table_stride, s.dtype) == (
        c.n_pages, 32, 2, 64, 1, 1, 1, 1)


def test_profiling_command_runs_them(capsys):
    from qweninferenceengine_b200.profiling import run_paged_q4

    run_paged_q4(3, 200, 16, 64, 2)
    out = capsys.readouterr().out
    for name in ("rope_append_paged_q4", "attention_paged_q4", "with weights", "evict_paged_q4", "expand_paged_q4"):
        assert name in out


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H,K,D,P,rot,inter", [
    (9, 3, 128, 64, 112, False), (7, 7, 64, 16, 48, False), (2, 1, 64, 64, 32, False), (3, 1, 128, 256, 80, True),
    (6, 6, 128, 16, 32, False), (4, 1, 128, 16, 128, False), (9, 9, 64, 32, 64, True)])
def test_append_of_kv_heads_that_do_not_fill_a_cta(dtype, H, K, D, P, rot, inter):
    lens = [P + 3, 1, 0, 200, 77]
    c = ref.Cache(40, lens, H, K, D, P, dtype, kept=True)
    check_append(c, [P + 1, 1, 0, 150, 77], rot, inter, ragged=True, pad=3, far=4000)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_codes_of_narrow_groups_far_from_zero(dtype):
    """Groups whose least value is 1 to 16,000 steps from zero, of random values, of values on
    and beside the borders between two codes, and of two values."""
    n, D = 600, 128
    c = ref.Cache(41, [n], 2, 2, D, 64, dtype)
    v = c.randn(n, 2, D).double()
    away = 2.0 ** torch.linspace(-4, 14, n, device="cuda", dtype=torch.float64)[:, None, None]
    size = 2.0 ** (torch.arange(n, device="cuda") % 9 - 4).double()[:, None, None]
    sign = (1 - 2 * (torch.arange(n, device="cuda") % 2)).double()[:, None, None]
    v[::3] = torch.arange(D, device="cuda") % 31 / 2.0
    v[1::6] = (torch.arange(D, device="cuda") % 2).double()
    v = ((v + sign * away) * size).to(dtype)
    k = v.flip(0).contiguous()
    pool = c.pool.clone()
    ops.rope_append_paged_q4(c.handle(), c.randn(n, 2, D), k, v, c.seq_len, torch.zeros(D // 2, device="cuda"),
                             cu_tokens=ints(0, n))
    c.store(0, torch.arange(n, device="cuda"), k, v, pool=pool)
    a, b = ref.views(c.pool, D, dtype), ref.views(pool, D, dtype)
    for x, y in zip(a[:2], b[:2]):
        assert torch.equal(x, y)
    for x, y in zip(a[2:], b[2:]):   # (0 of either sign; NaN where nothing was written)
        assert torch.equal(torch.isnan(x), torch.isnan(y)) and torch.equal(x.nan_to_num(7.0), y.nan_to_num(7.0))


def test_attention_of_long_contexts_is_not_off_to_one_side():
    """Outputs near zero, whose parts (lows, steps times codes, the codes' bias) are not: what the
    sums lose must not add up.

    The mean error over a sequence's outputs.  A tile's four MMAs cut off at most 2^-23 of
    their sums each, together 2^-21 A of A = sum of weights (|low| + 31 step), codes with a
    bias of 16 being at most 31.  All else errs to both sides: the output's rounding, u |out|
    at most, and the additions of the T tiles, 2^-24 A each, so that the mean of N such
    errors is within 6 of its deviations, 6 sqrt((u^2 mean(out^2) + T 2^-48 A^2) / N)."""
    n, L, H, K, D = 12, 16384, 32, 8, 128
    c = ref.Cache(50, [L] * n, H, K, D, 64, F16)
    out = ops.attention_paged_q4(c.handle(), c.q, c.seq_len)[3].double()
    slots = c.all_slots(3)
    k, v = c.rows(3, slots)
    page, block, r = c.place(3, slots)
    step, low = ref.views(c.pool, D, F16)[3][page, :, block, :, r].double().abs().unbind(-1)   # [L, K, D / 32]
    want, size = [], []
    for h in range(K):
        w = torch.softmax(c.q[3, h * 4: h * 4 + 4].double() @ k[:, h].T * D ** -0.5, -1)
        want.append(w @ v[:, h])
        size.append((w @ (low + 31 * step)[:, h]).amax())
    want, A = torch.cat(want), torch.stack(size).amax().item()
    off = (out - want).mean().abs().item()
    both = (2.0 ** -22 * want.pow(2).mean().item() + L / 128 * 2.0 ** -48 * A ** 2) / want.numel()
    assert off <= 2.0 ** -21 * A + 6 * both ** 0.5, (off, A)
