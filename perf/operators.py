"""Measured cases of the paged-cache operators: rotation and append, decode
attention over pages, attention of a batch with a shared prefix, and attention
over the pages that a bound on their scores selects.

A case is a dict of sizes.  prepare() makes its inputs on the GPU from a seed,
run() is one pass: elementary torch operations where `own` is false, the
framework's operators where it is true.
"""
import math
import random

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def _case(name, op, dtype, n_seq, heads, kv_heads, head_dim, page, length, **more):
    return dict(name=name, op=op, dtype=dtype, n_seq=n_seq, heads=heads, kv_heads=kv_heads,
                head_dim=head_dim, page=page, length=length, **more)


def listed():
    return [
        # one new token of one sequence: the batch-1 decode step's rotation and cache write
        _case("append_decode_1", "append", "f16", 1, 12, 2, 128, 16, 512, new=1, hnd=False,
              interleaved=False, rotary=128),
        # one new token of each of 256 sequences, the largest batch of a decode step
        _case("append_decode_256", "append", "bf16", 256, 12, 2, 128, 64, 300, new=1, hnd=True,
              interleaved=False, rotary=128),
        # a prompt chunk of ragged prompts behind cached turns (odd lengths, some with nothing new)
        _case("append_prompts", "append", "f16", 17, 12, 2, 128, 64, 1500, new=1024, hnd=False,
              interleaved=False, rotary=128),
        # two long prompts, interleaved pairs, a quarter of each head not rotated
        _case("append_long_interleaved", "append", "bf16", 2, 32, 8, 128, 256, 8704, new=8191,
              hnd=False, interleaved=True, rotary=96),
        # batch-1 decode at the benchmark's context
        _case("paged_1x512", "paged", "f16", 1, 12, 2, 128, 16, 512, hnd=False),
        # a decode step of 64 sequences of unequal lengths
        _case("paged_64x2048", "paged", "bf16", 64, 12, 2, 128, 64, 2048, hnd=False),
        # small heads in small pages, head-major pages
        _case("paged_33x1777_d64", "paged", "f16", 33, 16, 8, 64, 16, 1777, hnd=True),
        # a few requests behind one system prompt
        _case("prefix_8x1000", "prefix", "f16", 8, 12, 2, 128, 16, 70, hnd=False, prefix=1000),
        # a full batch behind a long document
        _case("prefix_64x8704", "prefix", "bf16", 64, 32, 8, 128, 64, 300, hnd=False, prefix=8704),
        # many samples of one very long prompt: the largest
        _case("prefix_256x32768", "prefix", "f16", 256, 12, 2, 128, 128, 257, hnd=False,
              prefix=32768),
        # one long context, a sixteenth of its pages
        _case("sparse_1x32768", "sparse", "f16", 1, 12, 2, 128, 64, 32768, hnd=False, select=32),
        # a batch of very long contexts
        _case("sparse_16x131072", "sparse", "bf16", 16, 32, 8, 128, 64, 131072, hnd=False,
              select=96),
    ]


def _spread(rng, low, high):
    """A whole number spread evenly over the logarithm of low .. high."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["append", "paged", "prefix", "sparse"])
    heads, kv_heads, head_dim = rng.choice(
        [(12, 2, 128), (32, 8, 128), (16, 8, 64), (14, 2, 64), (8, 8, 128), (16, 1, 128), (24, 2, 64)])
    c = dict(op=op, dtype=rng.choice(["f16", "bf16"]), heads=heads, kv_heads=kv_heads,
             head_dim=head_dim, page=rng.choice([16, 32, 64, 128, 256]), hnd=rng.random() < 0.3)
    if op == "append":
        if rng.random() < 0.4:
            c.update(n_seq=_spread(rng, 1, 256), length=_spread(rng, 1, 400), new=1)
        else:
            c.update(n_seq=_spread(rng, 1, 24), new=_spread(rng, 2, 1200))
            c["length"] = c["new"] + rng.randrange(0, 700)
        c.update(interleaved=rng.random() < 0.3,
                 rotary=head_dim if rng.random() < 0.7 else head_dim // 2)
    elif op == "paged":
        c["n_seq"] = _spread(rng, 1, 128)
        c["length"] = _spread(rng, 1, max(2, min(65536, 150000 // c["n_seq"])))
    elif op == "prefix":
        c["n_seq"] = _spread(rng, 1, 256)
        c["length"] = rng.randrange(0, 300)
        c["prefix"] = _spread(rng, 1, max(2, min(65536, 2000000 // c["n_seq"])))
    else:
        c["n_seq"] = _spread(rng, 1, 24)
        c["length"] = _spread(rng, 64, max(128, min(131072, 1000000 // c["n_seq"])))
        c["select"] = rng.randrange(4, 97)
    return c


def _lengths(c):
    """(positions of each sequence, new tokens of each): unequal, one or two
    sequences of a larger batch with a single position or none."""
    rng = random.Random(c["n_seq"] * 7919 + c["length"])
    n, top = c["n_seq"], c["length"]
    lens = [top] + [rng.randint((top + 3) // 4, top) for _ in range(n - 1)]
    if n >= 4 and top >= 1:
        lens[2] = 1
    if n >= 8:
        lens[5] = 0
    if c["op"] != "append":
        return lens, [0] * n
    if c["new"] == 1:
        return lens, [min(1, x) for x in lens]
    new = [min(x, c["new"] if i == 0 else rng.randint(1, c["new"])) for i, x in enumerate(lens)]
    if n >= 6:
        new[3] = 0
    return lens, new


def _pages(x, page):
    return -(-x // page)


def _randn(shape, gen, dtype):
    out = torch.empty(shape, dtype=dtype, device="cuda")
    return out.normal_(generator=gen)


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[c["dtype"]]
    n, H, K, D, P = c["n_seq"], c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    lens, new = _lengths(c)
    prefix = c.get("prefix", 0)
    width = max(1, _pages(max(lens), P))
    n_prefix = _pages(prefix, P)
    n_pages = n * width + n_prefix + 3
    order = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
    shape = (n_pages, K, P, D) if c["hnd"] else (n_pages, P, K, D)
    k_pages, v_pages = _randn(shape, gen, dtype), _randn(shape, gen, dtype)
    if c["hnd"]:
        k_pages, v_pages = k_pages.transpose(1, 2), v_pages.transpose(1, 2)
    s = dict(case=c, op=c["op"], k_pages=k_pages, v_pages=v_pages,
             table=order[: n * width].view(n, width).contiguous(),
             seq_len=torch.tensor(lens, dtype=torch.int32, device="cuda"), scale=1 / math.sqrt(D))
    if c["op"] in ("append", "sparse"):
        # what the cache holds before the call: each page's least and largest keys
        s["bounds"] = torch.zeros((n_pages, 2, K, D), dtype=dtype, device="cuda")
        at = torch.arange(width * P, device="cuda").view(width, P, 1, 1)
        for i in range(n):
            there, ids = at < lens[i] - new[i], s["table"][i].long()
            keys = k_pages[ids]
            if c["op"] == "sparse":  # pages unlike one another, as topics of a text are
                keys = keys * 0.5 + _randn((width, 1, K, D), gen, dtype)
                k_pages[ids] = keys
            s["bounds"][ids, 0] = torch.where(there, keys, math.inf).amin(1)
            s["bounds"][ids, 1] = torch.where(there, keys, -math.inf).amax(1)
    if c["op"] == "append":
        rows = sum(new) + (5 if c["new"] > 1 else 0)  # a padded chunk: rows behind the last sequence
        rows = n if c["new"] == 1 else rows
        qkv = _randn((rows, (H + 2 * K) * D), gen, dtype)  # one projection's output
        s["q"] = qkv[:, : H * D].view(rows, H, D)
        s["k"] = qkv[:, H * D : (H + K) * D].view(rows, K, D)
        s["v"] = qkv[:, (H + K) * D :].view(rows, K, D)
        s["q_out"] = torch.zeros((rows, H, D), dtype=dtype, device="cuda")
        R = c["rotary"]
        s["inv_freq"] = torch.tensor([1e6 ** (-2 * i / R) for i in range(R // 2)],
                                     dtype=torch.float32, device="cuda")
        s["cu_tokens"] = None
        if c["new"] > 1:
            cu = [0]
            for x in new:
                cu.append(cu[-1] + x)
            s["cu_tokens"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
        # which sequence and position each row is, for the plain form (-1: none)
        if c["new"] == 1:
            row = [(i if x else -1, x - 1) for i, x in enumerate(lens)]
        else:
            row = [(i, lens[i] - new[i] + j) for i in range(n) for j in range(new[i])]
        s["live"] = torch.tensor([i for i, r in enumerate(row) if r[0] >= 0], device="cuda")
        s["row_seq"] = torch.tensor([r[0] for r in row if r[0] >= 0], device="cuda")
        s["row_pos"] = torch.tensor([r[1] for r in row if r[0] >= 0], device="cuda")
    else:
        s["q"] = _randn((n, H, D), gen, dtype)
    if c["op"] == "prefix":
        s["prefix_pages"] = order[n * width : n * width + n_prefix].contiguous()
        s["prefix_len"] = prefix
    if c["op"] == "sparse":
        s["select"] = c["select"]
    return s


# --------------------------------------------------------------- plain form --
def _rotate(x, cos, sin, rotary, interleaved):
    x, rest = x[..., :rotary].float(), x[..., rotary:]
    cos, sin = cos[:, None], sin[:, None]
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        y = torch.stack((a * cos - b * sin, a * sin + b * cos), dim=-1).flatten(-2)
    else:
        a, b = x.chunk(2, dim=-1)
        y = torch.cat((a * cos - b * sin, a * sin + b * cos), dim=-1)
    return torch.cat((y.to(rest.dtype), rest), dim=-1)


def _append_plain(s):
    c, live = s["case"], s["live"]
    P, K, D = c["page"], c["kv_heads"], c["head_dim"]
    angle = s["row_pos"].double()[:, None] * s["inv_freq"].double()  # far positions: 64 bits
    cos, sin = angle.cos().float(), angle.sin().float()
    s["q_out"][live] = _rotate(s["q"][live], cos, sin, c["rotary"], c["interleaved"])
    k = _rotate(s["k"][live], cos, sin, c["rotary"], c["interleaved"])
    page, slot = s["table"][s["row_seq"], s["row_pos"] // P].long(), s["row_pos"] % P
    s["k_pages"][page, slot] = k
    s["v_pages"][page, slot] = s["v"][live]
    lo, hi = s["bounds"][:, 0].float(), s["bounds"][:, 1].float()
    first = (slot == 0)[:, None, None].expand(-1, K, D)  # a page begun anew forgets its old bounds
    at = page[:, None, None].expand(-1, K, D)
    key = k.float()
    inf = torch.full_like(key, math.inf)
    lo = lo.scatter_reduce(0, at, torch.where(first, inf, -inf), "amax")
    hi = hi.scatter_reduce(0, at, torch.where(first, -inf, inf), "amin")
    s["bounds"][:, 0] = lo.scatter_reduce(0, at, key, "amin").to(k.dtype)
    s["bounds"][:, 1] = hi.scatter_reduce(0, at, key, "amax").to(k.dtype)
    return dict(q=s["q_out"], k=s["k_pages"], v=s["v_pages"], bounds=s["bounds"])


def _join(scores, values, dtype):
    """Softmax over the last axis of the scores together, and its sum of the
    values; (out [n, heads, d], lse).  A row of -inf alone gives zeros."""
    top = torch.stack([x.amax(-1) for x in scores]).amax(0).clamp(min=-1e30)
    weight = [torch.exp(x - top[..., None]) for x in scores]
    total = torch.stack([w.sum(-1) for w in weight]).sum(0)
    out = torch.stack([values_of(w) for w, values_of in zip(weight, values)]).sum(0)
    out = out / torch.where(total > 0, total, 1.0)[..., None]
    return out.flatten(1, 2).to(dtype), (top + total.log()).flatten(1, 2)


def _grouped(s):
    c = s["case"]
    q = s["q"].float() * s["scale"]
    return q.view(c["n_seq"], c["kv_heads"], c["heads"] // c["kv_heads"], c["head_dim"])


def _own_pages(s):
    """Scores and values of each sequence's own pages."""
    table = s["table"].long()
    k, v = (s[x][table].flatten(1, 2).float() for x in ("k_pages", "v_pages"))
    score = torch.einsum("bhgd,blhd->bhgl", _grouped(s), k)
    there = torch.arange(k.shape[1], device=k.device) < s["seq_len"][:, None]
    score = score.masked_fill(~there[:, None, None], -math.inf)
    return score, lambda w: torch.einsum("bhgl,blhd->bhgd", w, v)


def _paged_plain(s):
    score, values = _own_pages(s)
    out, lse = _join([score], [values], s["q"].dtype)
    return dict(out=out, lse=lse)


def _prefix_plain(s):
    score, values = _own_pages(s)
    ids = s["prefix_pages"].long()
    k, v = (s[x][ids].flatten(0, 1)[: s["prefix_len"]].float() for x in ("k_pages", "v_pages"))
    shared = torch.einsum("bhgd,lhd->bhgl", _grouped(s), k)
    out, lse = _join([shared, score],
                     [lambda w: torch.einsum("bhgl,lhd->bhgd", w, v), values], s["q"].dtype)
    return dict(out=out, lse=lse)


def _sparse_plain(s):
    c, table = s["case"], s["table"].long()
    n, K, P, S = c["n_seq"], c["kv_heads"], c["page"], s["select"]
    G, width = c["heads"] // K, table.shape[1]
    q = s["q"].double().view(n, K, G, -1)  # pages next to the border: 64 bits
    bounds = s["bounds"][table].double()
    score = torch.einsum("bhd,bnhd->bhn", q.clamp(min=0).sum(2), bounds[:, :, 1])
    score += torch.einsum("bhd,bnhd->bhn", q.clamp(max=0).sum(2), bounds[:, :, 0])
    at = torch.arange(width, device=score.device)
    have = ((s["seq_len"] + P - 1) // P)[:, None]
    score = score.masked_fill(((at < 1) | (at == have - 1))[:, None], math.inf)
    score = score.masked_fill((at >= have)[:, None], -math.inf)
    best = score.sort(dim=-1, descending=True, stable=True).indices[..., :S]
    best = torch.where(best < have[:, None], best, width).sort(-1).values
    best = torch.cat((best, best.new_full((n, K, max(0, S - width)), width)), dim=-1)
    listed_there = best < width
    page = torch.gather(table[:, None].expand(-1, K, -1), 2, best.clamp(max=width - 1))
    head = torch.arange(K, device=page.device)[None, :, None]
    k, v = (s[x].transpose(1, 2)[page, head].flatten(2, 3).float() for x in ("k_pages", "v_pages"))
    score = torch.einsum("bhgd,bhld->bhgl", _grouped(s), k)
    pos = best[..., None] * P + torch.arange(P, device=best.device)
    there = (listed_there[..., None] & (pos < s["seq_len"][:, None, None, None])).flatten(2)
    score = score.masked_fill(~there[:, :, None], -math.inf)
    out, lse = _join([score], [lambda w: torch.einsum("bhgl,bhld->bhgd", w, v)], s["q"].dtype)
    pages = torch.where(listed_there, best, -1).to(torch.int32)
    return dict(pages=pages, out=out, lse=lse)


# ------------------------------------------------------ the framework's calls --
def _run_own(s):
    from qweninferenceengine_b200 import ops

    kv = ops.PagedKV(s["k_pages"], s["v_pages"], s["table"], s.get("bounds"))
    if s["op"] == "append":
        q = ops.rope_append_paged(kv, s["q"], s["k"], s["v"], s["seq_len"], s["inv_freq"],
                                  cu_tokens=s["cu_tokens"], interleaved=s["case"]["interleaved"],
                                  out=s["q_out"])
        return dict(q=q, k=s["k_pages"], v=s["v_pages"], bounds=s["bounds"])
    if s["op"] == "paged":
        out, lse = ops.attention_paged(kv, s["q"], s["seq_len"], scale=s["scale"], return_lse=True)
        return dict(out=out, lse=lse)
    if s["op"] == "prefix":
        out, lse = ops.attention_prefix_paged(kv, s["q"], s["seq_len"], s["prefix_pages"],
                                              s["prefix_len"], scale=s["scale"], return_lse=True)
        return dict(out=out, lse=lse)
    pages = ops.select_pages(kv, s["q"], s["seq_len"], s["select"], n_first=1, n_last=1)
    out, lse = ops.attention_sparse_paged(kv, s["q"], s["seq_len"], pages, scale=s["scale"],
                                          return_lse=True)
    return dict(pages=pages, out=out, lse=lse)


def run(state):
    if own:
        return _run_own(state)
    return {"append": _append_plain, "paged": _paged_plain, "prefix": _prefix_plain,
            "sparse": _sparse_plain}[state["op"]](state)


# ------------------------------------------------------------------- work ----
def work(case):
    c = case
    n, H, K, D, P = c["n_seq"], c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    lens, new = _lengths(c)
    live = sum(x > 0 for x in lens)
    if c["op"] == "append":
        tokens = sum(new)
        begun = sum(_pages(x, P) - (x - y) // P for x, y in zip(lens, new) if y)
        return dict(bytes=2.0 * (2 * tokens * (H + 2 * K) * D + 2 * 2 * begun * K * D)
                    + 4 * (c["rotary"] // 2 + n + begun),
                    flops=3.0 * tokens * (H + K) * c["rotary"])
    small = 2.0 * 2 * n * H * D + 4 * n * H + 4 * n  # q, out, lse, lengths
    if c["op"] == "sparse":
        S = c["select"]
        held = sum(_pages(x, P) for x in lens)
        kept = sum(min(x, S * P) for x in lens)
        ranked = sum(_pages(x, P) for x in lens if _pages(x, P) > S)
        return dict(bytes=small + 2.0 * 2 * kept * K * D + 2.0 * 2 * ranked * K * D
                    + 4 * held + 4 * n * K * S,
                    flops=4.0 * kept * H * D + 4.0 * ranked * K * D)
    own_positions, prefix = sum(lens), c.get("prefix", 0)
    table = 4 * (sum(_pages(x, P) for x in lens) + _pages(prefix, P))
    if c["op"] == "prefix":
        live = n
    return dict(bytes=small + 2.0 * 2 * (own_positions + prefix) * K * D + table,
                flops=4.0 * H * D * (own_positions + prefix * live))


# ------------------------------------------- the definition, in 64 bits -------
def _exact_append(s):
    c = s["case"]
    R, P = c["rotary"], c["page"]
    q, k, v, bounds = (s[x].double() for x in ("q_out", "k_pages", "v_pages", "bounds"))
    angle = torch.outer(s["row_pos"].double(), s["inv_freq"].double())
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    half = R // 2

    def spun(x):
        x = x[s["live"]].double()
        if c["interleaved"]:
            z = torch.view_as_complex(x[..., :R].reshape(*x.shape[:-1], half, 2).contiguous()) * turn
            x[..., :R] = torch.view_as_real(z).reshape(*x.shape[:-1], R)
        else:
            z = torch.complex(x[..., :half].contiguous(), x[..., half:R].contiguous()) * turn
            x[..., :half], x[..., half:R] = z.real, z.imag
        return x

    q[s["live"]] = spun(s["q"])
    key = spun(s["k"])
    place = s["table"][s["row_seq"], s["row_pos"] // P].long() * P + s["row_pos"] % P
    k[place // P, place % P] = key
    v[place // P, place % P] = s["v"][s["live"]].double()
    lens, new = _lengths(c)
    for i in range(c["n_seq"]):
        for j in range((lens[i] - new[i]) // P, _pages(lens[i], P) if new[i] else 0):
            held = k[s["table"][i, j].item(), : min(P, lens[i] - j * P)]
            bounds[s["table"][i, j].item(), 0] = held.amin(0)
            bounds[s["table"][i, j].item(), 1] = held.amax(0)
    return dict(q=q, k=k, v=v, bounds=bounds)


def _exact_rows(s, i, pages, length, shared):
    """Output and lse of sequence i over the positions of `pages` (one list for
    each kv head, or one for all) below `length`, and the shared prefix."""
    c = s["case"]
    P, K = c["page"], c["kv_heads"]
    G = c["heads"] // K
    outs, lses = [], []
    for h in range(K):
        logical = pages[h] if isinstance(pages, list) else pages
        at = (logical[:, None] * P + torch.arange(P, device="cuda")).flatten()
        ids = s["table"][i][logical].long()
        keep = at < length
        k = s["k_pages"][ids, :, h].flatten(0, 1)[keep].double()
        v = s["v_pages"][ids, :, h].flatten(0, 1)[keep].double()
        if shared is not None:
            k, v = torch.cat((shared[0][:, h], k)), torch.cat((shared[1][:, h], v))
        q = s["q"][i, h * G : (h + 1) * G].double()
        x = q @ k.T * s["scale"]
        lses.append(torch.logsumexp(x, -1) if x.shape[1] else x.new_full((G,), -math.inf))
        outs.append(torch.softmax(x, -1) @ v if x.shape[1] else torch.zeros_like(q))
    return torch.cat(outs), torch.cat(lses)


def _exact_list(s, i, length):
    """The pages of sequence i that each kv head takes, ascending."""
    c = s["case"]
    K, P, S = c["kv_heads"], c["page"], s["select"]
    have = _pages(length, P)
    everything = torch.arange(have, device="cuda")
    if have <= S:
        return [everything] * K
    b = s["bounds"][s["table"][i, :have].long()].double()
    q = s["q"][i].double().view(K, -1, c["head_dim"])
    taken = []
    for h in range(K):
        x = q[h][:, None]
        score = torch.maximum(x * b[:, 0, h], x * b[:, 1, h]).sum((0, 2)).tolist()
        middle = sorted(range(1, have - 1), key=lambda p: (-score[p], p))[: S - 2]
        taken.append(torch.tensor(sorted([0, have - 1] + middle), device="cuda"))
    return taken


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["op"] == "append":
        return _exact_append(s)
    lens, _ = _lengths(c)
    shared = None
    if c["op"] == "prefix":
        ids = s["prefix_pages"].long()
        shared = [s[x][ids].flatten(0, 1)[: s["prefix_len"]].double() for x in ("k_pages", "v_pages")]
    outs, lses, lists = [], [], []
    for i, length in enumerate(lens):
        pages = torch.arange(_pages(length, c["page"]), device="cuda")
        if c["op"] == "sparse":
            pages = _exact_list(s, i, length)
            row = torch.full((c["kv_heads"], s["select"]), -1, device="cuda")
            for h, x in enumerate(pages):
                row[h, : len(x)] = x
            lists.append(row)
        out, lse = _exact_rows(s, i, pages, length, shared)
        outs.append(out)
        lses.append(lse)
    got = dict(out=torch.stack(outs), lse=torch.stack(lses))
    return dict(pages=torch.stack(lists), **got) if c["op"] == "sparse" else got
