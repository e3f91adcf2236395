"""The operators over a 4-bit paged cache against their formulas in 64 bits
(paged_q4_reference.py, which also derives the tolerances)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import paged_q4_reference as ref  # noqa: E402
import paged_reference  # noqa: E402
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


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def freqs(rot):
    return torch.tensor([1e6 ** (-2 * i / rot) for i in range(rot // 2)], dtype=torch.float32, device="cuda")


# ------------------------------------------------------------------ append ---
def rotate_exact(x, angle, rot, interleaved):
    y = x.double().clone()
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    one, two = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    x1, x2 = x[..., one].double(), x[..., two].double()
    y[..., one], y[..., two] = x1 * c - x2 * s, x1 * s + x2 * c
    return y


def check_append(c, new, rot, interleaved, ragged, axes=1, pad=0, in_place=False, far=0, given=True):
    """Appends the last `new` slots of each sequence and checks every byte of the pool, the
    kept weights and positions, and q."""
    n, H, K, D = len(c.lens), c.heads, c.kv_heads, c.dim
    past = [x - y for x, y in zip(c.lens, new)]
    rows = sum(new) + pad if ragged else n
    qkv = c.randn(rows, (H + 2 * K) * D)
    q, k, v = (x.view(rows, -1, D) for x in qkv.split([H * D, K * D, K * D], dim=1))
    cu = None
    if ragged:
        cu = [0]
        for x in new:
            cu.append(cu[-1] + x)
        row = [(i, past[i] + j) for i in range(n) for j in range(new[i])] + [None] * pad
        cu = ints(*cu)
    else:
        row = [(i, past[i]) if new[i] else None for i in range(n)]
    live = [r for r, x in enumerate(row) if x is not None]
    slots = torch.tensor([row[r][1] for r in live], device="cuda")
    inv = freqs(rot)
    pos = torch.randint(-far, far + 1, (axes, rows), generator=c.g, device="cuda").to(torch.int32)
    which = torch.randint(0, axes, (rot // 2,), generator=c.g, device="cuda").to(torch.uint8)
    at = pos[:, live].double() if given else slots.double()[None]
    angle = at.t()[:, which.long()] * inv.double() if axes > 1 else at[0][:, None] * inv.double()
    pool, q_in = c.pool.clone(), q.clone()
    weights, positions = (None, None) if c.weights is None else (c.weights.clone(), c.positions.clone())
    out = q if in_place else torch.full((rows, H, D), 7.0, dtype=c.dtype, device="cuda")
    got = ops.rope_append_paged_q4(c.handle(), q, k, v, c.seq_len, inv, cu_tokens=cu,
                                   positions=(pos if axes > 1 else pos[0]) if given else None,
                                   pair_axis=which if axes > 1 else None, interleaved=interleaved, out=out)
    assert got is out
    u = paged_reference.U[c.dtype]
    y = rotate_exact(q_in[live], angle, rot, interleaved)
    # sine and cosine rounded to fp32, two products, their sum: half a step each
    err = 4 * 2.0 ** -24 * torch.full_like(y, 2.0) * q_in[live].double().abs().amax()
    assert ((out[live].double() - y).abs() - (u * y.abs() + 2 * err + 1e-7)).max().item() <= 0
    rest = [r for r in range(rows) if r not in set(live)]
    if rest:
        assert (out[rest] == (q_in[rest] if in_place else 7.0)).all()
    turned = ref.to_type(rotate_exact(k[live], angle, rot, interleaved), c.dtype)
    for j, r in enumerate(live):
        i, slot = row[r]
        c.store(i, torch.tensor([slot], device="cuda"), turned[j: j + 1], v[r: r + 1], pool=pool)
        if weights is not None:
            weights[i, :, slot] = 0
            positions[i, :, slot] = pos[0, r] if given else slot
    assert torch.equal(c.pool, pool)
    if weights is not None:
        assert torch.equal(c.weights, weights) and torch.equal(c.positions, positions)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,K,D,P,rot,inter,axes", [
    (12, 2, 128, 16, 128, False, 1), (32, 8, 128, 64, 96, True, 3), (14, 2, 64, 256, 64, False, 2),
    (8, 8, 64, 32, 16, True, 1), (16, 1, 128, 128, 64, False, 4), (3, 3, 64, 16, 48, False, 3)])
def test_append_one_token(dtype, H, K, D, P, rot, inter, axes):
    lens = [1, P, P + 1, 2 * P - 1, 0, 3 * P, 300]
    c = ref.Cache(1, lens, H, K, D, P, dtype, kept=True)
    check_append(c, [min(x, 1) for x in lens], rot, inter, ragged=False, axes=axes, far=5000)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,K,D,P,rot,inter,axes", [
    (12, 2, 128, 16, 128, False, 1), (12, 2, 128, 64, 128, False, 3), (32, 8, 128, 256, 96, True, 1),
    (14, 2, 64, 128, 64, False, 2), (8, 8, 64, 32, 32, True, 3), (5, 5, 128, 16, 16, False, 1)])
def test_append_ragged(dtype, H, K, D, P, rot, inter, axes):
    lens = [1, P, P + 1, 2 * P - 1, 0, 3 * P, 300, 517, 64, 5]
    new = [1, P, 1, P, 0, 2 * P + 1, 300, 100, 0, 2]
    c = ref.Cache(2, lens, H, K, D, P, dtype, kept=axes > 1, head_gap=1)
    check_append(c, new, rot, inter, ragged=True, axes=axes, pad=5, far=3000)


def test_append_at_slots_in_place_and_far_positions():
    c = ref.Cache(3, [70, 200], 12, 2, 128, 64, F16, kept=True)
    check_append(c, [70, 133], 128, False, ragged=True, given=False, in_place=True)
    c = ref.Cache(4, [70, 33], 12, 2, 128, 64, F16)
    check_append(c, [70, 33], 128, False, ragged=True, far=2 ** 31 - 1)
    c = ref.Cache(5, [2111], 12, 2, 128, 64, BF16)
    check_append(c, [2100], 128, False, ragged=True, far=200000)


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_groups_at_the_borders_of_their_type(dtype):
    """Groups of one value, of the type's extremes, of subnormals, with values on the borders
    between two codes, with an infinity or NaN."""
    top = torch.finfo(dtype).max
    tiny = 2.0 ** -24 if dtype is F16 else 2.0 ** -133
    c = ref.Cache(6, [40], 4, 2, 128, 16, dtype)
    rows = torch.zeros(40, 2, 128, dtype=torch.float64)
    rows[0] = 3.25
    rows[1, :, ::2], rows[1, :, 1::2] = top, -top
    rows[2] = torch.arange(128) % 32 * tiny
    rows[3] = torch.arange(128) % 31 / 2          # 0 .. 15: codes at k / 2
    rows[4] = (torch.arange(128) % 31 / 2 - 8) * 0.375
    rows[5] = torch.randn(2, 128)
    rows[5, 0, 7], rows[5, 1, 40], rows[5, 0, 127] = math.nan, math.inf, -math.inf
    rows[6] = -0.0
    rows[7] = torch.arange(128) % 2 * tiny
    rows[8, :, 0] = 1.0
    rows[9] = top
    rows[9, :, 5] = top / 2
    rows[10] = 1.0 + torch.arange(128) % 16 * torch.finfo(dtype).eps
    for r in range(11, 40):
        rows[r] = torch.randn(2, 128) * 10.0 ** (r % 7 - 3)
    v = rows.to(device="cuda").to(dtype)
    k = v.flip(0).contiguous()
    q = c.randn(40, 4, 128)
    pool = c.pool.clone()
    got = ops.rope_append_paged_q4(c.handle(), q, k, v, c.seq_len, torch.zeros(64, device="cuda"),
                                   cu_tokens=ints(0, 40))
    assert torch.equal(got, q)   # angles of 0
    # (turned by angles of 0: an infinity's mate is NaN, 0 times one)
    k = ref.to_type(rotate_exact(k, torch.zeros(40, 64, device="cuda").double(), 128, False), dtype)
    c.store(0, torch.arange(40, device="cuda"), k, v, pool=pool)
    a, b = ref.views(c.pool, 128, dtype), ref.views(pool, 128, dtype)
    for x, y in zip(a[:2], b[:2]):
        assert torch.equal(x, y)
    for x, y in zip(a[2:], b[2:]):   # (any NaN, and 0 of either sign)
        assert torch.equal(torch.isnan(x), torch.isnan(y)) and torch.equal(x.nan_to_num(7.0), y.nan_to_num(7.0))


# --------------------------------------------------------------- attention ---
LENS = [1, 15, 16, 17, 0, 63, 64, 65, 300, 513]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("H,K,D,P", [(12, 2, 128, 16), (32, 8, 128, 64), (14, 2, 64, 256), (8, 8, 64, 32),
                                     (16, 1, 128, 128), (3, 3, 128, 64), (24, 2, 64, 16), (64, 1, 128, 64),
                                     (40, 2, 64, 64)])
def test_attention(dtype, kept, H, K, D, P):
    c = ref.Cache(10, LENS, H, K, D, P, dtype, kept=kept)
    before = c.weights.clone() if kept else None
    scale = D ** -0.5
    out, lse = ops.attention_paged_q4(c.handle(), c.q, c.seq_len, return_lse=True)
    r = ref.attention(c, scale)
    ref.check_attention((out, lse), r)
    if kept:
        ref.check_weights(c.weights, before, r)
    again = ops.attention_paged_q4(c.handle(), c.q, c.seq_len, scale=scale)
    assert torch.equal(again, out)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,H,K,D,P", [([9001], 12, 2, 128, 64), ([20011, 3], 16, 8, 64, 16),
                                          ([700] * 70, 12, 2, 128, 256), ([5000, 0, 1, 4097], 32, 8, 128, 128)])
def test_attention_long_and_many(dtype, lens, H, K, D, P):
    c = ref.Cache(11, lens, H, K, D, P, dtype, kept=True)
    before = c.weights.clone()
    got = ops.attention_paged_q4(c.handle(), c.q, c.seq_len, return_lse=True)
    r = ref.attention(c, D ** -0.5)
    ref.check_attention(got, r)
    ref.check_weights(c.weights, before, r)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_of_large_scores_and_values(dtype):
    """Scores of hundreds, heavy rows at both ends, steps that differ by 2^20 and values near
    the type's ends."""
    c = ref.Cache(12, [600, 77], 12, 2, 128, 64, dtype, kept=True)
    big = 60000.0 if dtype is F16 else 1e30
    slots = c.all_slots(0)
    k, v = c.randn(600, 2, 128), c.randn(600, 2, 128)
    k[5], k[599] = k[5] * 8, k[599] * 8
    v[::7] = v[::7] * 2.0 ** -10
    v[3] = v[3] * 1000
    c.store(0, slots, k, v)
    k2, v2 = c.randn(77, 2, 128), c.randn(77, 2, 128)
    v2[:, :, ::3] = big
    v2[:, :, 1::3] = -big
    c.store(1, c.all_slots(1), k2, v2)
    c.q[0] *= 6
    before = c.weights.clone()
    got = ops.attention_paged_q4(c.handle(), c.q, c.seq_len, scale=1.0, return_lse=True)
    r = ref.attention(c, 1.0)
    ref.check_attention(got, r)
    ref.check_weights(c.weights, before, r)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_of_queries_at_their_types_ends(dtype):
    """Tiny and huge queries beside small ones in one head, and heads of zeros."""
    c = ref.Cache(13, [130], 12, 2, 128, 64, dtype)
    c.q[0, 0] *= 2.0 ** -20 if dtype is F16 else 2.0 ** -100
    c.q[0, 1] = 0
    c.q[0, 2, :64] *= 2.0 ** 12
    c.q[0, 3] = 2.0 ** 15 * (1 + c.q[0, 3] / 100)
    for scale in (1.0, -0.05, 0.0):
        got = ops.attention_paged_q4(c.handle(), c.q, c.seq_len, scale=scale, return_lse=True)
        ref.check_attention(got, ref.attention(c, scale))


def test_attention_nan_and_infinite_groups():
    """A key with a NaN group makes its head's outputs NaN, a value's group its 32 elements;
    others, and slots behind the end, do not notice."""
    for dtype in DTYPES:
        c = ref.Cache(14, [100, 100, 31], 12, 2, 128, 16, dtype, kept=True)
        k, v = c.randn(100, 2, 128), c.randn(100, 2, 128)
        k[40, 0, 3] = math.nan
        v[41, 1, 70] = math.inf
        c.store(0, c.all_slots(0), k, v)
        out, lse = ops.attention_paged_q4(c.handle(), c.q, c.seq_len, return_lse=True)
        bad = torch.zeros_like(out, dtype=torch.bool)
        bad[0, :6] = True
        bad[0, 6:, 64:96] = True
        assert torch.equal(torch.isnan(out), bad) and torch.isfinite(out[~bad]).all()
        assert torch.isnan(lse[0, :6]).all() and torch.isfinite(lse[0, 6:]).all() and torch.isfinite(lse[1:]).all()
        assert torch.isnan(c.weights[0, 0, :100]).all() and torch.isfinite(c.weights[0, 0, 100:]).all()
        assert torch.isfinite(c.weights[0, 1]).all() and torch.isfinite(c.weights[1:]).all()
        clean = ref.attention(c, 128 ** -0.5)
        off = (out.double() - clean[0]).abs() - clean[3] - 1e-7
        assert off[~bad].max().item() <= 0


def test_attention_in_place_strided_and_without_positions():
    c = ref.Cache(15, [65, 0, 130], 12, 2, 128, 64, BF16, head_gap=2)
    want = ref.attention(c, 128 ** -0.5)
    wide = torch.zeros(3, 2 * 12 * 128 + 8, dtype=BF16, device="cuda")
    q = wide[:, 8: 8 + 1536].view(3, 12, 128)
    q.copy_(c.q)
    out = wide[:, 8 + 1536:].view(3, 12, 128)
    ops.attention_paged_q4(c.handle(), q, c.seq_len, out=out)
    ref.check_attention((out, None), want)
    got = ops.attention_paged_q4(c.handle(), q, c.seq_len, out=q, return_lse=True)
    ref.check_attention(got, want)
    kept = ref.Cache(15, [65, 0, 130], 12, 2, 128, 64, BF16, kept=True)
    before, want = kept.weights.clone(), ref.attention(kept, 128 ** -0.5)
    ref.check_attention(ops.attention_paged_q4(kept.handle(), kept.q, kept.seq_len, out=kept.q, return_lse=True), want)
    ref.check_weights(kept.weights, before, want)
    none = ref.Cache(16, [0, 0], 12, 2, 64, 16, F16, kept=True)
    before = none.weights.clone()
    out, lse = ops.attention_paged_q4(none.handle(), none.q, none.seq_len, return_lse=True)
    assert (out == 0).all() and torch.isneginf(lse).all() and torch.equal(none.weights, before)


# ------------------------------------------------------------------ expand ---
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K,D,P", [(2, 128, 16), (8, 128, 64), (2, 64, 256), (1, 64, 32), (3, 128, 128)])
def test_expand(dtype, K, D, P):
    lens = [1, P, P + 1, 0, 300, 5]
    c = ref.Cache(20, lens, 2 * K, K, D, P, dtype)
    take = [1, P, 3, 0, 299, 5]
    cu = ints(*[sum(take[:i]) for i in range(len(take) + 1)])
    n = sum(take) + 4
    k, v = (torch.full((n, K + 1, D), 7.0, dtype=dtype, device="cuda")[:, :K] for _ in range(2))
    got = ops.expand_paged_q4(c.handle(), c.seq_len, cu, out=(k, v))
    assert got[0] is k and got[1] is v
    at = 0
    for i, m in enumerate(take):
        for x, y in zip((k, v), c.rows(i, c.all_slots(i)[lens[i] - m:])):
            assert torch.equal(x[at: at + m], ref.to_type(y, dtype))
        at += m
    assert (k[at:] == 7.0).all() and (v[at:] == 7.0).all()
    k, v = ops.expand_paged_q4(c.handle(), c.seq_len, cu, n_rows=sum(take))
    assert k.shape == (sum(take), K, D)
    full = torch.full((2, len(lens), K, D), 7.0, dtype=dtype, device="cuda")
    ops.expand_paged_q4(c.handle(), c.seq_len, out=(full[0], full[1]))
    for i, x in enumerate(lens):
        if x:
            assert torch.equal(full[0, i], ref.to_type(c.rows(i, c.all_slots(i)[-1:])[0][0], dtype))
        else:
            assert (full[:, i] == 7.0).all()


# ------------------------------------------------------------------- evict ---
def check_evict(c, n_keep, n_first, n_recent, out=None):
    before = c.pool.clone()
    parts = ref.views(before, c.dim, c.dtype)
    weights, positions = c.weights.clone(), c.positions.clone()
    w, p = weights.tolist(), positions.tolist()
    got = ops.evict_paged_q4(c.handle(), c.seq_len, n_keep, n_first, n_recent, out=out)
    assert got.tolist() == [min(x, n_keep) for x in c.lens]
    for i, x in enumerate(c.lens):
        for h in range(c.kv_heads):
            pairs = ref.evict(w[i][h], p[i][h], x, n_keep, n_first, n_recent)
            if not pairs:
                continue
            to, src = (torch.tensor(t, device="cuda") for t in zip(*pairs))
            tp, tb, tr = c.place(i, to)
            sp, sb, sr = c.place(i, src)
            for part in parts:
                part[tp, h, tb, :, tr] = part[sp, h, sb, :, sr]
            weights[i, h, to], positions[i, h, to] = weights[i, h, src], positions[i, h, src]
    assert torch.equal(c.pool, before)
    assert torch.equal(c.weights.nan_to_num(-3.0), weights.nan_to_num(-3.0)) and torch.equal(c.positions, positions)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K,D,P,keep,first,recent", [
    (2, 128, 16, 64, 4, 16), (8, 128, 64, 256, 0, 0), (2, 64, 256, 100, 10, 50), (1, 64, 32, 1, 0, 1),
    (3, 128, 128, 511, 1, 300), (2, 128, 64, 17, 17, 0)])
def test_evict(dtype, K, D, P, keep, first, recent):
    lens = [1, keep, keep + 1, 0, 300, 513, 2 * keep, 1025]
    c = ref.Cache(30, lens, 2 * K, K, D, P, dtype, kept=True)
    for i, x in enumerate(lens):   # slots in no order, as earlier evictions leave them
        if x:
            order = torch.randperm(x, generator=c.g, device="cuda").to(torch.int32)
            c.positions[i, :, :x] = order * 3
    check_evict(c, keep, first, recent)


def test_evict_ties_nan_and_signs():
    """Equal weights (the lower slot stays), NaN, infinities, negative weights, zeros of
    either sign; more guarded slots than are kept."""
    c = ref.Cache(31, [200, 200, 200, 200, 2000], 4, 2, 64, 16, F16, kept=True)
    c.weights[0] = 1.0
    c.weights[1] = torch.randint(0, 4, c.weights[1].shape, generator=c.g, device="cuda").float()
    c.weights[2, :, ::5] = math.nan
    c.weights[2, :, 1::5] = math.inf
    c.weights[2, :, 2::5] = -math.inf
    c.weights[3, :, ::2] = -0.0
    c.weights[3, :, 1::2] = 0.0
    c.weights[3, :, 50:60] = -1.0
    c.weights[3, :, 60:70] = 1e-42
    c.weights[4] = torch.randint(0, 3, c.weights[4].shape, generator=c.g, device="cuda").float() - 1
    for keep, first, recent in ((100, 0, 0), (50, 5, 20), (30, 100, 100), (30, 0, 2 ** 30), (199, 2 ** 30, 0)):
        check_evict(c, keep, first, recent)   # (of the same lengths again: slots behind are candidates)


def test_evict_positions_at_their_types_ends_and_lengths_in_place():
    c = ref.Cache(32, [90, 20, 64], 2, 1, 128, 32, BF16, kept=True)
    c.positions[0, :, :90] = torch.linspace(-2 ** 31, 2 ** 31 - 1, 90, dtype=torch.float64, device="cuda").to(torch.int32)
    check_evict(c, 40, 2 ** 30, 2 ** 30, out=c.seq_len)
    assert c.seq_len.tolist() == [40, 20, 40]


def test_evict_a_long_row():
    c = ref.Cache(33, [70000, 33000], 2, 1, 64, 256, F16, kept=True)
    check_evict(c, 2500, 4, 600)
    c = ref.Cache(34, [40000], 2, 2, 64, 256, F16, kept=True)
    check_evict(c, 39000, 4, 600)


# ----------------------------------------------------------- used together ---
@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_under_a_budget(dtype):
    """A prompt, then steps of append, attention and eviction; what is kept is followed in
    64 bits from the same cache."""
    H, K, D, P, keep = 12, 2, 128, 16, 48
    lens = [47, 90, 0, 1]
    n = len(lens)
    c = ref.Cache(40, [0] * n, H, K, D, P, dtype, width=8, kept=True)
    inv = freqs(D)
    seen = list(lens)
    kv = c.handle()
    x = c.randn(sum(lens), H + 2 * K, D)
    cu = ints(*[sum(lens[:i]) for i in range(n + 1)])
    seq_len = ints(*lens)
    pos = torch.cat([torch.arange(m, device="cuda") for m in lens]).to(torch.int32)
    ops.rope_append_paged_q4(kv, x[:, :H], x[:, H: H + K], x[:, H + K:], seq_len, inv, cu_tokens=cu, positions=pos)
    c.lens, c.seq_len = list(lens), seq_len
    for i, m in enumerate(lens):
        assert (c.weights[i, :, :m] == 0).all()
        assert torch.equal(c.positions[i, 0, :m].cpu(), torch.arange(m, dtype=torch.int32))
    for step in range(4):
        check_evict(c, keep, 2, 10, out=c.seq_len)
        c.lens = [min(m, keep) for m in c.lens]
        seq_len += 1
        c.lens = [m + 1 for m in c.lens]
        x = c.randn(n, H + 2 * K, D)
        q = ops.rope_append_paged_q4(kv, x[:, :H], x[:, H: H + K], x[:, H + K:], seq_len, inv, positions=ints(*seen))
        for i in range(n):
            assert (c.positions[i, :, c.lens[i] - 1] == seen[i]).all() and (c.weights[i, :, c.lens[i] - 1] == 0).all()
        seen = [m + 1 for m in seen]
        before = c.weights.clone()
        got = ops.attention_paged_q4(kv, q, seq_len, return_lse=True)
        r = ref.attention(c, D ** -0.5, q=q)
        ref.check_attention(got, r)
        ref.check_weights(c.weights, before, r)
    # the newest positions are still there
    for i in range(n):
        for h in range(K):
            held = set(c.positions[i, h, : c.lens[i]].tolist())
            assert {s for s in range(max(0, seen[i] - 10), seen[i])} <= held


def test_a_step_captured_and_replayed():
    H, K, D, P = 12, 2, 128, 64
    c = ref.Cache(41, [100, 333, 64], H, K, D, P, F16, width=8, kept=True)
    kv, inv = c.handle(), freqs(D)
    x = c.randn(3, H + 2 * K, D)
    pos = ints(99, 500, 63)
    out, q = torch.zeros(3, H, D, dtype=F16, device="cuda"), torch.zeros(3, H, D, dtype=F16, device="cuda")
    new_len, cu = ints(0, 0, 0), ints(0, 60, 120, 180)
    rows = torch.zeros(2, 180, K, D, dtype=F16, device="cuda")

    def step():
        ops.rope_append_paged_q4(kv, x[:, :H], x[:, H: H + K], x[:, H + K:], c.seq_len, inv, positions=pos, out=q)
        ops.attention_paged_q4(kv, q, c.seq_len, out=out)
        ops.evict_paged_q4(kv, c.seq_len, 60, 4, 16, out=new_len)
        ops.expand_paged_q4(kv, new_len, cu, out=(rows[0], rows[1]))

    state = [t.clone() for t in (c.pool, c.weights, c.positions)]

    def restore():
        for t, old in zip((c.pool, c.weights, c.positions), state):
            t.copy_(old)

    step()
    want = [t.clone() for t in (out, q, new_len, rows, c.pool, c.weights, c.positions)]
    restore()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    for _ in range(3):
        restore()
        for t in (out, q, new_len, rows):
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for t, w in zip((out, q, new_len, rows, c.pool, c.weights, c.positions), want):
            assert torch.equal(t, w)


def test_two_streams_at_once():
    caches = [ref.Cache(50 + i, [3000 + 17 * i, 40], 12, 2, 128, 64, F16, kept=True) for i in range(2)]
    want, before = [], []
    for c in caches:
        before.append(c.weights.clone())
        want.append(ops.attention_paged_q4(c.handle(), c.q, c.seq_len))
        c.weights.copy_(before[-1])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in caches]
    got = [[], []]
    for _ in range(5):
        for i, c in enumerate(caches):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.attention_paged_q4(c.handle(), c.q, c.seq_len))
    torch.cuda.synchronize()
    for i, c in enumerate(caches):
        assert all(torch.equal(x, want[i]) for x in got[i])
        r = ref.attention(c, 128 ** -0.5)
        off = (c.weights.double() - before[i].double() - 5 * r[2]).abs() - 5 * r[5] - 2.0 ** -20 * (before[i] + 5 * r[2])
        assert off.max().item() <= 0


# ---------------------------------------------------- what the device sees ---
def reported(text):
    assert status() == QWEN_ERR_INVALID_ARGUMENT
    assert text in lib().qwen_last_error().decode()


def test_lengths_beyond_the_table():
    """That sequence is left as it was, the others are served."""
    c = ref.Cache(60, [40, 64, 30], 12, 2, 128, 16, F16, kept=True)
    kv, inv = c.handle(), freqs(128)
    long = ints(40, 65, 30)
    want = ref.attention(c, 128 ** -0.5)
    out = torch.full((3, 12, 128), 7.0, dtype=F16, device="cuda")
    before = c.weights.clone()
    ops.attention_paged_q4(kv, c.q, long, out=out)
    reported("out-of-range")
    assert (out[1] == 7.0).all() and torch.equal(c.weights[1], before[1])
    out[1], before[1] = want[0][1].half(), c.weights[1] - want[2][1]
    ref.check_attention((out, None), want)
    pool = c.pool.clone()
    x = c.randn(3, 16, 128)
    q = torch.full((3, 12, 128), 7.0, dtype=F16, device="cuda")
    ops.rope_append_paged_q4(kv, x[:, :12], x[:, 12:14], x[:, 14:], long, inv, out=q)
    reported("out-of-range")
    assert (q[1] == 7.0).all() and not (q[0] == 7.0).any()
    own = [int(t) for t in c.table[1]]
    assert torch.equal(c.pool[own], pool[own])
    new_len, w, p = ints(-5, -5, -5), c.weights[1].clone(), c.positions[1].clone()
    ops.evict_paged_q4(kv, long, 20, 1, 1, out=new_len)
    reported("out-of-range")
    assert new_len.tolist() == [20, -5, 20] and torch.equal(c.weights[1], w) and torch.equal(c.positions[1], p)
    k, v = (torch.full((3, 2, 128), 7.0, dtype=F16, device="cuda") for _ in range(2))
    ops.expand_paged_q4(kv, long, out=(k, v))
    reported("out-of-range")
    assert (k[1] == 7.0).all() and (v[1] == 7.0).all() and not (k[0] == 7.0).any()


def test_pages_outside_the_pool():
    """Nothing is read or written there; the positions are left out."""
    c = ref.Cache(61, [100, 64], 12, 2, 128, 16, F16, kept=True)
    kv = c.handle()
    keep = [s for s in range(100) if not 32 <= s < 48]
    short = ref.Cache(61, [100, 64], 12, 2, 128, 16, F16, kept=True)
    k, v = c.rows(0, torch.tensor(keep, device="cuda"))
    for bad in (-1, c.n_pages, 2 ** 31 - 1):
        c.table[0, 2] = bad
        out, lse = ops.attention_paged_q4(kv, c.q, c.seq_len, return_lse=True)
        reported("out-of-range")
        for h in range(12):
            s = (c.q[0, h].double() @ k[:, h // 6].T) * 128 ** -0.5
            assert abs(lse[0, h].item() - torch.logsumexp(s, -1).item()) < 1e-4
            assert (out[0, h].double() - torch.softmax(s, -1) @ v[:, h // 6]).abs().max().item() < 4e-3
        ref.check_attention((out[1:], lse[1:]), tuple(x[1:] for x in ref.attention(short, 128 ** -0.5)))
        rows = ops.expand_paged_q4(kv, c.seq_len, ints(0, 100, 100), out=tuple(
            torch.full((100, 2, 128), 7.0, dtype=F16, device="cuda") for _ in range(2)))
        reported("out-of-range")
        assert (rows[0][32:48] == 7.0).all() and torch.equal(rows[0][keep], ref.to_type(k, F16))
        pool = c.pool.clone()
        x = c.randn(100, 16, 128)
        ops.rope_append_paged_q4(kv, x[:, :12], x[:, 12:14], x[:, 14:], c.seq_len, freqs(128), cu_tokens=ints(0, 100, 100))
        reported("out-of-range")
        own = {int(t) for i, t in enumerate(c.table[0]) if i != 2}
        others = [t for t in range(c.n_pages) if t not in own]
        assert torch.equal(c.pool[others], pool[others])
        c.pool.copy_(pool)
        c.weights[0, :, 36:40] = -1.0   # of that page: to be filled from behind
        ops.evict_paged_q4(kv, ints(100, 40), 40, 0, 0)   # (the other sequence has no more)
        reported("out-of-range")
        assert torch.equal(c.pool[others], pool[others])
        c.pool.copy_(pool)


def test_rows_out_of_order_and_axes_beyond():
    c = ref.Cache(62, [40, 30], 4, 2, 64, 16, F16)
    kv = c.handle()
    pool = c.pool.clone()
    x = c.randn(20, 8, 64)
    for cu in (ints(0, 41, 20), ints(5, 3, 20), ints(0, 10, 21), ints(-1, -1, -1)):
        ops.rope_append_paged_q4(kv, x[:, :4], x[:, 4:6], x[:, 6:], ints(0, 0), freqs(64), cu_tokens=cu)
        reported("out-of-range")
        ops.expand_paged_q4(kv, ints(0, 0), cu, n_rows=20)
        reported("out-of-range")
    assert torch.equal(c.pool, pool)
    pos = torch.zeros(2, 20, dtype=torch.int32, device="cuda")
    ops.rope_append_paged_q4(kv, x[:, :4], x[:, 4:6], x[:, 6:], c.seq_len, freqs(64), cu_tokens=ints(0, 10, 20),
                             positions=pos, pair_axis=torch.full((32,), 2, dtype=torch.uint8, device="cuda"))
    reported("out-of-range")


def test_refusals_of_the_wrappers():
    c = ref.Cache(63, [40, 30], 4, 2, 64, 16, F16, kept=True)
    kv = c.handle()
    x = c.randn(2, 8, 64)
    q, k, v = x[:, :4], x[:, 4:6], x[:, 6:]
    inv = freqs(64)
    with pytest.raises(ValueError):
        ops.PagedKVQ4(c.pool, c.table, torch.float32)
    with pytest.raises(ValueError):
        ops.PagedKVQ4(c.pool[..., :-1], c.table, F16)
    with pytest.raises(ValueError):
        ops.PagedKVQ4(c.pool, c.table, F16, weights=c.weights[:, :, :-1])
    with pytest.raises(ValueError):
        ops.PagedKVQ4(c.pool, c.table, F16, positions=c.weights)
    with pytest.raises(ValueError):
        ops.rope_append_paged_q4(kv, q, k, v, c.seq_len, inv, positions=ints(1, 2, 3))
    with pytest.raises(ValueError):
        ops.rope_append_paged_q4(kv, q, k, v, c.seq_len, inv, positions=ints(1, 2).long())
    with pytest.raises(ValueError):
        ops.rope_append_paged_q4(kv, q, k, v, c.seq_len, inv, pair_axis=torch.zeros(31, dtype=torch.uint8, device="cuda"))
    with pytest.raises(QwenError):   # two axes and no pair_axis
        ops.rope_append_paged_q4(kv, q, k, v, c.seq_len, inv, positions=torch.zeros(2, 2, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        ops.attention_paged_q4(kv, c.q.to(BF16), c.seq_len)
    with pytest.raises(ValueError):
        ops.expand_paged_q4(kv, c.seq_len, ints(0, 1, 2))
    with pytest.raises(ValueError):
        ops.evict_paged_q4(kv, c.seq_len, 0)
    with pytest.raises(ValueError):
        ops.evict_paged_q4(kv, c.seq_len, 1 << 32)
    with pytest.raises(QwenError):
        ops.evict_paged_q4(kv, c.seq_len, 1 << 25)
    with pytest.raises(QwenError):
        ops.evict_paged_q4(ops.PagedKVQ4(c.pool, c.table, F16), c.seq_len, 10)
