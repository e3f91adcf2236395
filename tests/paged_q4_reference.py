"""The operators over a 4-bit paged cache in 64 bits, and the bounds that the tests hold
the kernels to."""
import math

import torch

from paged_reference import U

F16, BF16 = torch.float16, torch.bfloat16


def to_type(x, dtype):
    """64-bit values rounded to fp32 and then to the cache's type."""
    return x.float().to(dtype)


def quantise(x):
    """(codes uint8, step, low) of rows [..., d] of a 16-bit type: codes [..., d / 32, 32]."""
    g = x.unflatten(-1, (-1, 32)).double()
    bad = ~torch.isfinite(g).all(-1)
    low, high = g.amin(-1), g.amax(-1)
    step = to_type((high - low) / 15, x.dtype)
    nan = torch.tensor(math.nan, dtype=x.dtype, device=x.device)
    step, low = torch.where(bad, nan, step), torch.where(bad, nan, low.to(x.dtype))
    s = step.double()[..., None]
    code = torch.where(s > 0, torch.round((g - low.double()[..., None]) / s), 0.0)
    return code.nan_to_num(0.0).clamp(0, 15).to(torch.uint8), step, low


def views(pool, dim, dtype):
    """(key codes, value codes) [page, head, block, group, slot, 16] and (steps and lows of
    keys, of values) [page, head, block, group, slot, 2] of a pool."""
    G = dim // 32
    kc, vc = (pool[..., a: a + 8 * dim].unflatten(-1, (G, 16, 16)) for a in (0, 8 * dim))
    ks, vs = (pool[..., a: a + 2 * dim].view(dtype).unflatten(-1, (G, 16, 2)) for a in (16 * dim, 18 * dim))
    return kc, vc, ks, vs


class Cache:
    """A pool of random rows.  What no sequence's slots cover is filled with ones: codes of
    15 and NaN for step and low, so that a slot that takes part in a result by mistake
    shows."""

    def __init__(self, seed, lens, heads, kv_heads, dim, page, dtype, spare=3, width=None, kept=False,
                 device="cuda", head_gap=0):
        self.g = torch.Generator(device=device).manual_seed(seed)
        self.lens, self.heads, self.kv_heads, self.dim, self.page = list(lens), heads, kv_heads, dim, page
        self.dtype, self.device = dtype, device
        n = len(lens)
        self.width = width or max(1, max((-(-x // page) for x in lens), default=1))
        self.n_pages = n * self.width + spare
        order = torch.randperm(self.n_pages, generator=self.g, device=device).to(torch.int32)
        self.table = order[: n * self.width].view(n, self.width).contiguous()
        whole = torch.full((self.n_pages, kv_heads + head_gap, page // 16, 20 * dim), 255, dtype=torch.uint8,
                           device=device)
        self.pool = whole[:, :kv_heads]
        self.cap = self.width * page
        self.seq_len = torch.tensor(self.lens, dtype=torch.int32, device=device)
        self.weights = self.positions = None
        if kept:
            self.weights = torch.rand((n, kv_heads, self.cap), generator=self.g, device=device)
            self.positions = torch.arange(self.cap, dtype=torch.int32, device=device).expand(
                n, kv_heads, -1).contiguous()
        for i, x in enumerate(self.lens):
            self.store(i, torch.arange(x, device=device), self.randn(x, kv_heads, dim),
                       self.randn(x, kv_heads, dim))
        self.q = self.randn(n, heads, dim)

    def randn(self, *shape):
        return torch.randn(shape, generator=self.g, device=self.device).to(self.dtype)

    def place(self, i, slots):
        return self.table[i, slots // self.page].long(), slots % self.page // 16, slots % 16

    def store(self, i, slots, k, v, pool=None):
        """Quantises rows k, v [n, kv_heads, d] into slots of sequence i."""
        if not len(slots):
            return
        page, block, r = self.place(i, slots)
        kc, vc, ks, vs = views(self.pool if pool is None else pool, self.dim, self.dtype)
        for x, c, s in ((k, kc, ks), (v, vc, vs)):
            code, step, low = quantise(x)
            c[page, :, block, :, r] = code[..., 0::2] | code[..., 1::2] << 4
            s[page, :, block, :, r] = torch.stack((step, low), -1)

    def rows(self, i, slots):
        """Keys and values of slots of sequence i, in 64 bits: [n, kv_heads, d]."""
        page, block, r = self.place(i, slots)
        got = []
        kc, vc, ks, vs = views(self.pool, self.dim, self.dtype)
        for c, s in ((kc, ks), (vc, vs)):
            byte, p = c[page, :, block, :, r], s[page, :, block, :, r].double()
            code = torch.stack((byte & 15, byte >> 4), -1).flatten(-2).double()
            got.append((p[..., 1:] + code * p[..., :1]).flatten(-2))
        return got

    def sizes(self, i, slots):
        """|low| + code step of the same: what rounding errors are relative to."""
        page, block, r = self.place(i, slots)
        got = []
        kc, vc, ks, vs = views(self.pool, self.dim, self.dtype)
        for c, s in ((kc, ks), (vc, vs)):
            byte, p = c[page, :, block, :, r], s[page, :, block, :, r].double()
            code = torch.stack((byte & 15, byte >> 4), -1).flatten(-2).double()
            got.append((p[..., 1:].abs() + code * p[..., :1]).flatten(-2))
        return got

    def all_slots(self, i):
        return torch.arange(self.lens[i], device=self.device)

    def handle(self, **kept):
        from qweninferenceengine_b200 import ops

        kept = kept or dict(weights=self.weights, positions=self.positions)
        return ops.PagedKVQ4(self.pool, self.table, self.dtype, **kept)


def attention(c, scale, q=None, lens=None):
    """(out, lse, weights [n, kv_heads, cap] that the query heads give, and bounds on the
    errors of the three) in 64 bits.

    The bounds.  A score is a sum of 2 D products (q with codes times steps, q with lows)
    in fp32, off by at most 2^-23 (2 D S) with S the sum of |q| (|low| + code step) times
    |scale|; with the scaling and the exponential a weight p is off, relatively, by d =
    2^-23 (2 D S + 16 + 2 max|s|).  Products of weights with values: a weight times a step
    is rounded to fp16 at most once (2^-11; to two values it is 2^-22), sums of L of them
    in fp32 are off by 2^-23 L; what they multiply is at most |low| + code step.  So
    |out error| <= A (2^-11 + 2 d + 2^-22 L) + u |out|, A = sum p (|low| + code step) / sum
    p; and where codes are multiplied with a bias of up to 128 beside them, that is taken off
    again, by weights times steps of 16 bits, 143 2^-17 sum p step / sum p.  |lse error| <= d + 2^-23 L + 2^-22 |lse|, and a weight exp(s - lse) is off by (d +
    the lse's) p, the sum of a group's by 2^-23 of it and of what it is added to."""
    q = c.q if q is None else q
    lens = c.lens if lens is None else lens
    n, H, D = q.shape
    K, G = c.kv_heads, H // c.kv_heads
    u, kind = U[c.dtype], dict(dtype=torch.float64, device=q.device)
    out, tol = torch.zeros((n, H, D), **kind), torch.zeros((n, H, D), **kind)
    lse, lse_tol = torch.full((n, H), -math.inf, **kind), torch.zeros((n, H), **kind)
    w_all, w_tol = torch.zeros((n, K, c.cap), **kind), torch.zeros((n, K, c.cap), **kind)
    for i in range(n):
        L = lens[i]
        if L == 0:
            continue
        slots = torch.arange(L, device=q.device)
        k, v = c.rows(i, slots)
        ka, va = c.sizes(i, slots)
        page, block, r = c.place(i, slots)
        vstep = views(c.pool, c.dim, c.dtype)[3][page, :, block, :, r][..., 0].double().repeat_interleave(32, -1)
        for h in range(K):
            rows = slice(h * G, (h + 1) * G)
            x = q[i, rows].double()
            s = x @ k[:, h].T * scale
            d = 2.0 ** -23 * (2 * D * (x.abs() @ ka[:, h].T * abs(scale)).amax(-1) + 16 + 2 * s.abs().amax(-1))
            w = torch.softmax(s, -1)
            out[i, rows] = w @ v[:, h]
            tol[i, rows] = (w @ va[:, h]) * (2.0 ** -11 + 2 * d + 2.0 ** -22 * L)[:, None] + u * out[i, rows].abs() + \
                143 * 2.0 ** -17 * (w @ vstep[:, h])
            lse[i, rows] = torch.logsumexp(s, -1)
            lse_tol[i, rows] = d + 2.0 ** -23 * L + 2.0 ** -22 * lse[i, rows].abs()
            w_all[i, h, :L] = w.sum(0)
            w_tol[i, h, :L] = (w * (d + lse_tol[i, rows])[:, None]).sum(0) + 2.0 ** -22 * w.sum(0)
    return out, lse, w_all, tol, lse_tol, w_tol


def check_attention(got, ref):
    out, lse = got
    want, want_lse, _, tol, lse_tol, _ = ref
    assert torch.isfinite(out).all()
    off = (out.double() - want).abs() - tol - 1e-7   # 1e-7: two steps of fp16's subnormals
    assert off.max().item() <= 0, (off.max().item(), torch.nonzero(off > 0)[:5].tolist())
    if lse is not None:
        none = torch.isinf(want_lse)
        assert torch.equal(torch.isneginf(lse), none)
        off = ((lse.double() - want_lse).abs() - lse_tol)[~none]
        assert off.numel() == 0 or off.max().item() <= 0, off.max().item()


def check_weights(got, before, ref):
    want = before.double() + ref[2]
    off = (got.double() - want).abs() - ref[5] - 2.0 ** -23 * want.abs()
    assert off.max().item() <= 0, (off.max().item(), torch.nonzero(off > 0)[:5].tolist())
    untouched = ref[2] == 0
    assert torch.equal(got[untouched], before[untouched])


def evict(weights, positions, length, n_keep, n_first, n_recent):
    """Of one (sequence, kv head): [(to, from), ...], from lists."""
    if length <= n_keep:
        return []
    newest = max(positions[:length])
    guarded = [positions[j] < n_first or positions[j] > newest - n_recent for j in range(length)]
    order = sorted(range(length), key=lambda j: (
        not guarded[j], not math.isnan(weights[j]), 0.0 if math.isnan(weights[j]) else -weights[j], j))
    kept = set(order[:n_keep])
    holes = [j for j in range(n_keep) if j not in kept]
    comes = [j for j in range(n_keep, length) if j in kept]
    assert len(holes) == len(comes)
    return list(zip(holes, comes))
