"""The paged-cache operators in 64 bits, one sequence at a time, and the bounds
that the tests hold the kernels to."""
import math

import torch

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}   # half a step, relative


class Cache:
    """Pools of random pages.  What no sequence's positions cover is NaN, so that a
    masked position that takes part in a result shows."""

    def __init__(self, seed, lens, heads, kv_heads, dim, page, dtype, hnd=False, prefix=0, spare=3,
                 width=None, device="cuda"):
        self.g = torch.Generator(device=device).manual_seed(seed)
        self.lens, self.heads, self.kv_heads, self.dim, self.page = lens, heads, kv_heads, dim, page
        self.dtype, self.device, self.prefix = dtype, device, prefix
        n = len(lens)
        self.width = width or max(1, max((-(-x // page) for x in lens), default=1))
        n_prefix = -(-prefix // page)
        self.n_pages = n * self.width + n_prefix + spare
        order = torch.randperm(self.n_pages, generator=self.g, device=device).to(torch.int32)
        self.table = order[: n * self.width].view(n, self.width).contiguous()
        self.prefix_pages = order[n * self.width: n * self.width + n_prefix].contiguous()
        shape = (self.n_pages, kv_heads, page, dim) if hnd else (self.n_pages, page, kv_heads, dim)
        self.k = torch.full(shape, math.nan, dtype=dtype, device=device)
        self.v = torch.full(shape, math.nan, dtype=dtype, device=device)
        if hnd:
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        for i, x in enumerate(lens):
            self.fill(self.table[i], x)
        self.fill(self.prefix_pages, prefix)
        self.seq_len = torch.tensor(lens, dtype=torch.int32, device=device)
        self.q = self.randn(n, heads, dim)
        self.bounds = None

    def randn(self, *shape):
        return torch.randn(shape, generator=self.g, device=self.device).to(self.dtype)

    def fill(self, pages, length):
        for j in range(-(-length // self.page)):
            m = min(self.page, length - j * self.page)
            p = int(pages[j])
            self.k[p, :m] = self.randn(m, self.kv_heads, self.dim)
            self.v[p, :m] = self.randn(m, self.kv_heads, self.dim)

    def make_bounds(self):
        """Bounds of the positions held; NaN for pages that hold none."""
        self.bounds = torch.full((self.n_pages, 2, self.kv_heads, self.dim), math.nan,
                                 dtype=self.dtype, device=self.device)
        for i, x in enumerate(self.lens):
            for j in range(-(-x // self.page)):
                p = int(self.table[i, j])
                held = self.k[p, : min(self.page, x - j * self.page)]
                self.bounds[p, 0], self.bounds[p, 1] = held.amin(0), held.amax(0)
        return self.bounds

    def handle(self):
        from qweninferenceengine_b200 import ops

        return ops.PagedKV(self.k, self.v, self.table, self.bounds)

    def positions(self, i, h, columns=None):
        """Keys and values of kv head h that sequence i attends, in 64 bits."""
        ks, vs = [], []
        for j in range(-(-self.prefix // self.page)):
            p, m = int(self.prefix_pages[j]), min(self.page, self.prefix - j * self.page)
            ks.append(self.k[p, :m, h])
            vs.append(self.v[p, :m, h])
        if columns is None:
            columns = range(-(-self.lens[i] // self.page))
        for j in columns:
            if j < 0 or j * self.page >= self.lens[i]:
                continue
            p, m = int(self.table[i, j]), min(self.page, self.lens[i] - j * self.page)
            ks.append(self.k[p, :m, h])
            vs.append(self.v[p, :m, h])
        empty = torch.empty((0, self.dim), dtype=torch.float64, device=self.device)
        return (torch.cat([empty] + [x.double() for x in ks]),
                torch.cat([empty] + [x.double() for x in vs]))


def attention(cache, scale, lists=None, q=None):
    """(out, lse, bound on |out error|, bound on |lse error|) in 64 bits.

    The bounds.  u: half a step of the type.  A weight p = exp(s - m) is formed from
    a score that D products were added to in fp32 (a step of 2^-23 each, were they
    truncated), then scaled and exponentiated (a few steps): a relative error of at
    most d = 2^-23 (D S + 16 + 2 max|s|), S the largest sum of |q k| times the scale.
    Its product with v is taken after one rounding to the type (u); the L products
    and weights are added in fp32 (2^-23 L each).  So |out error| <= A (u + 2 d +
    2^-22 L) + u |out| with A = sum p |v| / sum p, and |lse error| <= d + 2^-23 L +
    2^-22 |lse|."""
    q = cache.q if q is None else q
    n, H, D = q.shape
    G = H // cache.kv_heads
    u = U[cache.dtype]
    out = torch.zeros((n, H, D), dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    lse = torch.full((n, H), -math.inf, dtype=torch.float64, device=q.device)
    lse_tol = torch.zeros_like(lse)
    for i in range(n):
        for h in range(cache.kv_heads):
            k, v = cache.positions(i, h, None if lists is None else lists[i][h].tolist())
            if k.shape[0] == 0:
                continue
            rows = slice(h * G, (h + 1) * G)
            x = q[i, rows].double()
            s = x @ k.T * scale
            d = 2.0 ** -23 * (D * (x.abs() @ k.abs().T * abs(scale)).amax(-1) + 16 + 2 * s.abs().amax(-1))
            w = torch.softmax(s, -1)
            out[i, rows] = w @ v
            L = k.shape[0]
            tol[i, rows] = (w @ v.abs()) * (u + 2 * d + 2.0 ** -22 * L)[:, None] + u * out[i, rows].abs()
            lse[i, rows] = torch.logsumexp(s, -1)
            lse_tol[i, rows] = d + 2.0 ** -23 * L + 2.0 ** -22 * lse[i, rows].abs()
    return out, lse, tol, lse_tol


def assert_attention(got, ref):
    out, lse = got
    want, want_lse, tol, lse_tol = ref
    assert torch.isfinite(out).all()
    off = (out.double() - want).abs() - tol - 1e-7   # 1e-7: two steps of fp16's subnormals
    assert off.max().item() <= 0, (off.max().item(), torch.nonzero(off > 0)[:5].tolist())
    none = torch.isinf(want_lse)
    assert torch.equal(torch.isneginf(lse), none)
    off = ((lse.double() - want_lse).abs() - lse_tol)[~none]
    assert off.numel() == 0 or off.max().item() <= 0, off.max().item()


def scores(cache, i):
    """Page scores [kv_heads, pages] of sequence i, from the definition."""
    n = -(-cache.lens[i] // cache.page)
    b = cache.bounds[cache.table[i, :n].long()].double()
    q = cache.q[i].double().view(cache.kv_heads, -1, 1, cache.dim)
    lo, hi = b[:, 0].permute(1, 0, 2)[:, None], b[:, 1].permute(1, 0, 2)[:, None]
    return torch.maximum(q * lo, q * hi).sum((1, 3))


def select(cache, n_select, n_first, n_last):
    out = torch.full((len(cache.lens), cache.kv_heads, n_select), -1, dtype=torch.int32)
    for i, x in enumerate(cache.lens):
        n = -(-x // cache.page)
        s = scores(cache, i).tolist() if n else None
        for h in range(cache.kv_heads):
            if n <= n_select:
                take = list(range(n))
            else:
                rank = lambda p: (-math.inf if math.isnan(s[h][p]) else -s[h][p], p)  # noqa: E731
                nan = [p for p in range(n_first, n - n_last) if math.isnan(s[h][p])]
                rest = [p for p in range(n_first, n - n_last) if not math.isnan(s[h][p])]
                best = (nan + sorted(rest, key=rank))[: n_select - n_first - n_last]
                take = sorted(list(range(n_first)) + best + list(range(n - n_last, n)))
            out[i, h, : len(take)] = torch.tensor(take, dtype=torch.int32)
    return out


def rotate(x, pos, inv_freq, interleaved):
    """(rotated rows in 64 bits, bound on the error before rounding): each of the two
    products and their sum is off by half a step of fp32, sin and cos by two steps
    each and by the fp32 angle after its reduction to turns (2^-24 2 pi)."""
    R = 2 * inv_freq.shape[0]
    a = pos.double()[:, None, None] * inv_freq.double()
    c, s = torch.cos(a), torch.sin(a)
    y = x.double().clone()
    one, two = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
    x1, x2 = x[..., one].double(), x[..., two].double()
    y[..., one], y[..., two] = x1 * c - x2 * s, x1 * s + x2 * c
    err = torch.zeros_like(y)
    err[..., one] = err[..., two] = (x1.abs() + x2.abs()) * 2.0 ** -24 * (2 * math.pi + 4 + 2)
    return y, err
