"""paged_reference.attention for whole batches behind a shared prefix at once (hundreds of
sequences one by one take minutes): the same formulas and bounds, in 64 bits."""
import math

import torch

from paged_reference import U


def attention(cache, scale):
    c = cache
    n, H, D = c.q.shape
    K, P = c.kv_heads, c.page
    G = H // K
    device = c.q.device
    at = torch.arange(c.width * P, device=device)
    there = torch.cat((torch.ones((n, c.prefix), dtype=torch.bool, device=device),
                       at < c.seq_len[:, None].to(device)), dim=1)[:, None]
    L = there.sum(-1).double()   # [n, 1]
    u = U[c.dtype]
    out, tol = (torch.zeros((n, H, D), dtype=torch.float64, device=device) for _ in range(2))
    lse, lse_tol = (torch.zeros((n, H), dtype=torch.float64, device=device) for _ in range(2))
    for h in range(K):
        shared = [x[c.prefix_pages.long(), :, h].flatten(0, 1)[: c.prefix].double() for x in (c.k, c.v)]
        own = [x[c.table.long(), :, h].flatten(1, 2).double() for x in (c.k, c.v)]
        own = [x.masked_fill(~(at < c.seq_len[:, None])[..., None], 0.0) for x in own]
        x = c.q[:, h * G:(h + 1) * G].double()

        def with_keys(y, f):   # y times all keys: [n, G, positions]
            return torch.cat((y @ f(shared[0]).T, y @ f(own[0]).transpose(1, 2)), dim=-1)

        def with_values(w, f):
            return w[..., : c.prefix] @ f(shared[1]) + w[..., c.prefix:] @ f(own[1])

        s = (with_keys(x, lambda k: k) * scale).masked_fill(~there, -math.inf)
        size = (with_keys(x.abs(), torch.abs) * abs(scale)).masked_fill(~there, 0.0).amax(-1)
        d = 2.0 ** -23 * (D * size + 16 + 2 * s.masked_fill(~there, 0.0).abs().amax(-1))
        w = torch.softmax(s, -1)
        w = torch.where(there, w, 0.0)   # (no position at all: NaN)
        rows = slice(h * G, (h + 1) * G)
        out[:, rows] = with_values(w, lambda v: v)
        tol[:, rows] = with_values(w, torch.abs) * (u + 2 * d + 2.0 ** -22 * L)[..., None] + u * out[:, rows].abs()
        lse[:, rows] = torch.logsumexp(s, -1)
        lse_tol[:, rows] = d + 2.0 ** -23 * L + 2.0 ** -22 * lse[:, rows].abs()
    none = torch.isinf(lse)
    return out, lse, tol, lse_tol.masked_fill(none, 0.0)
