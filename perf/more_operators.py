"""Measured cases of the operators over a paged cache held in 4 bits: rotation at given
positions and append, decode attention with and without accumulated weights,
reading rows back, eviction by accumulated weight.

A case is a dict of sizes.  prepare() makes its inputs on the GPU from a seed,
run() is one pass: elementary torch operations where `own` is false, the
framework's operators where it is true.

The cache: pool uint8 [n_pages, kv_heads, page / 16, 20 d].  A block of 16 slots is
key codes [d / 32][16][16 bytes], value codes the same, then the key groups'
(step, low) [d / 32][16][2] in the cache's type, and the value groups'.  Byte j of a
group of 32 elements holds element 2j in its low four bits and 2j + 1 in its high.
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
        # the batch-1 decode step of a layer: the new token appended, the cache attended
        _case("step_1x512", "step", "f16", 1, 12, 2, 128, 16, 512, axes=1, interleaved=False,
              rotary=128, weigh=False),
        # a decode step of 64 sequences with images among them (time, height, width), weights kept
        _case("step_64x2048_axes", "step", "bf16", 64, 12, 2, 128, 64, 2048, axes=3,
              interleaved=False, rotary=128, weigh=True),
        # small heads in small pages, weights kept
        _case("step_33x1777_d64", "step", "f16", 33, 16, 8, 64, 16, 1777, axes=1,
              interleaved=True, rotary=64, weigh=True),
        # one long context
        _case("attend_1x32768", "attend", "f16", 1, 12, 2, 128, 64, 32768, weigh=False),
        # a batch of long documents whose weights are kept, for a later eviction
        _case("attend_16x8704_weighed", "attend", "f16", 16, 32, 8, 128, 256, 8704, weigh=True),
        # the longest batch: the largest
        _case("attend_32x16384", "attend", "bf16", 32, 32, 8, 128, 64, 16384, weigh=False),
        # a chunk of ragged prompts behind cached turns (odd lengths, some with nothing new), read
        # back for the chunk's own attention
        _case("chunk_prompts", "chunk", "f16", 17, 12, 2, 128, 64, 1500, new=1024, axes=1,
              interleaved=False, rotary=128),
        # one prompt with an image, odd length
        _case("chunk_image", "chunk", "bf16", 1, 12, 2, 128, 16, 1201, new=1201, axes=3,
              interleaved=False, rotary=128),
        # two long prompts, interleaved pairs, a quarter of each head not rotated
        _case("chunk_long_interleaved", "chunk", "bf16", 2, 32, 8, 128, 256, 8704, new=8191,
              axes=1, interleaved=True, rotary=96),
        # a full batch some tokens over its budget, read back
        _case("evict_64x1060", "evict", "f16", 64, 12, 2, 128, 64, 1060, keep=1024),
        # one long prompt cut to a sixteenth
        _case("evict_1x32768", "evict", "bf16", 1, 12, 2, 128, 64, 32768, keep=2048),
        # long prompts of a batch cut to an eighth, small heads
        _case("evict_16x16384_d64", "evict", "f16", 16, 16, 8, 64, 16, 16384, keep=2047),
    ]


def _spread(rng, low, high):
    """A whole number spread evenly over the logarithm of low .. high."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["step", "attend", "chunk", "evict"])
    heads, kv_heads, head_dim = rng.choice(
        [(12, 2, 128), (32, 8, 128), (16, 8, 64), (14, 2, 64), (8, 8, 128), (16, 1, 128), (24, 2, 64)])
    c = dict(op=op, dtype=rng.choice(["f16", "bf16"]), heads=heads, kv_heads=kv_heads,
             head_dim=head_dim, page=rng.choice([16, 32, 64, 128, 256]))
    if op in ("step", "chunk"):
        c.update(axes=rng.choice([1, 1, 2, 3]), interleaved=rng.random() < 0.3,
                 rotary=head_dim if rng.random() < 0.7 else head_dim // 2)
    if op in ("step", "attend"):
        c["n_seq"] = _spread(rng, 1, 128)
        c["length"] = _spread(rng, 1, max(2, min(65536, 300000 // c["n_seq"])))
        c["weigh"] = rng.random() < 0.5
    elif op == "chunk":
        c.update(n_seq=_spread(rng, 1, 24), new=_spread(rng, 2, 1200))
        c["length"] = c["new"] + rng.randrange(0, 700)
    else:
        c["n_seq"] = _spread(rng, 1, 64)
        c["length"] = _spread(rng, 32, max(64, min(65536, 260000 // c["n_seq"])))
        c["keep"] = _spread(rng, 16, max(17, min(4096, c["length"])))
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
    if c["op"] != "chunk":
        return lens, [min(1, x) if c["op"] == "step" else 0 for x in lens]
    new = [min(x, c["new"] if i == 0 else rng.randint(1, c["new"])) for i, x in enumerate(lens)]
    if n >= 6:
        new[3] = 0
    return lens, new


def _pages(x, page):
    return -(-x // page)


def _randn(shape, gen, dtype):
    out = torch.empty(shape, dtype=dtype, device="cuda")
    return out.normal_(generator=gen)


# ---------------------------------------------------- the cache's layout ------
def _parts(pool, dim, dtype):
    """Views of a pool, or of pages of it: key and value codes [..., block, group, slot, 16] and
    (step, low) of keys and values [..., block, group, slot, 2]."""
    G = dim // 32
    codes = [pool[..., a * dim:(a + 8) * dim].unflatten(-1, (G, 16, 16)) for a in (0, 8)]
    steps = [pool[..., a * dim:(a + 2) * dim].view(dtype).unflatten(-1, (G, 16, 2)) for a in (16, 18)]
    return codes[0], codes[1], steps[0], steps[1]


def _quantised(x):
    """(codes as bytes [..., g, 16], (step, low) [..., g, 2]) of rows of whole groups."""
    y = x.unflatten(-1, (-1, 32)).double()  # values next to a border: 64 bits
    low, high = y.amin(-1, keepdim=True), y.amax(-1, keepdim=True)
    step = ((high - low) / 15).to(x.dtype).double()
    code = torch.where(step > 0, ((y - low) / step).round().clamp(max=15), 0.0).to(torch.uint8)
    return code[..., 0::2] | code[..., 1::2] << 4, torch.cat((step, low), -1).to(x.dtype)


def _values(codes, steps):
    """fp32 values [..., slot, d] of codes [..., group, slot, 16]."""
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float()
    x = steps[..., 1:].float() + code * steps[..., :1].float()
    return x.transpose(-3, -2).flatten(-2)


def _random_pool(shape, dim, gen, dtype):
    """Rows of normal values, quantised: their groups are drawn from 2^15 different ones."""
    pool = torch.empty(shape, dtype=torch.uint8, device="cuda")
    codes, steps = _quantised(_randn((1 << 15, 32), gen, dtype))
    kc, vc, ks, vs = _parts(pool, dim, dtype)
    for c, s in ((kc, ks), (vc, vs)):
        at = torch.randint(0, 1 << 15, c.shape[:-1], generator=gen, device="cuda")
        c.copy_(codes[at, 0])
        s.copy_(steps[at, 0])
    return pool


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[c["dtype"]]
    n, H, K, D, P = c["n_seq"], c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    lens, new = _lengths(c)
    width = max(1, _pages(max(lens), P))
    n_pages = n * width + 3
    order = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
    s = dict(case=c, op=c["op"], dtype=dtype, dim=D, scale=1 / math.sqrt(D),
             pool=_random_pool((n_pages, K, P // 16, 20 * D), D, gen, dtype),
             table=order[: n * width].view(n, width).contiguous(),
             seq_len=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    s["weights"] = s["positions"] = None
    if c.get("weigh") or c["op"] == "evict":
        # a few heavy slots, many light ones, as attention leaves them
        both = torch.empty((2, n, K, width * P), dtype=torch.float32, device="cuda")
        both[0] = _randn(both.shape[1:], gen, torch.float32).mul_(2).exp_()
        for i in range(n):  # what is cached: text in order, a tenth of it moved by earlier evictions
            at = torch.arange(width * P, device="cuda").expand(K, -1).clone()
            m = lens[i] // 10
            if m:
                at[:, lens[i] // 3:][:, :m] = at[:, lens[i] // 3:][:, :m].flip(-1)
            both[1, i] = at.to(torch.int32).view(torch.float32)
        s["both"] = both
        s["weights"], s["positions"] = both[0], both[1].view(torch.int32)
    if c["op"] == "evict":
        s["before"] = both.clone()
        s["keep"], s["first"], s["recent"] = c["keep"], min(4, c["keep"] // 4), c["keep"] // 4
        left = [min(x, c["keep"]) for x in lens]
        s["rows"] = sum(left)
        s["cu"] = torch.tensor([0] + left, dtype=torch.int32, device="cuda").cumsum(0).to(torch.int32)
        row = [(i, j) for i in range(n) for j in range(left[i])]
    if c["op"] in ("step", "attend"):
        s["q"] = _randn((n, H, D), gen, dtype)
    if c["op"] == "chunk":
        row = [(i, j) for i in range(n) for j in range(lens[i])]
        s["rows"] = len(row)
        s["cu"] = torch.tensor([0] + lens, dtype=torch.int32, device="cuda").cumsum(0).to(torch.int32)
    if c["op"] in ("chunk", "evict"):  # which sequence and slot each row read back is
        s["row_seq"], s["row_slot"] = (torch.tensor([r[k] for r in row], device="cuda") for k in (0, 1))
    if c["op"] in ("step", "chunk"):
        step = c["op"] == "step"
        rows = n if step else sum(new) + 5  # a padded chunk: rows behind the last sequence
        qkv = _randn((rows, (H + 2 * K) * D), gen, dtype)  # one projection's output
        s["q"] = qkv[:, : H * D].view(rows, H, D)
        s["k"] = qkv[:, H * D: (H + K) * D].view(rows, K, D)
        s["v"] = qkv[:, (H + K) * D:].view(rows, K, D)
        s["q_out"] = torch.zeros((rows, H, D), dtype=dtype, device="cuda")
        R, axes = c["rotary"], c["axes"]
        s["inv_freq"] = torch.tensor([1e6 ** (-2 * i / R) for i in range(R // 2)],
                                     dtype=torch.float32, device="cuda")
        s["cu_tokens"] = None
        if step:
            tok = [(i, x - 1) for i, x in enumerate(lens) if x]
            live = [i for i, x in enumerate(lens) if x]
        else:
            tok = [(i, lens[i] - new[i] + j) for i in range(n) for j in range(new[i])]
            live = list(range(len(tok)))
            s["cu_tokens"] = torch.tensor([0] + new, dtype=torch.int32, device="cuda").cumsum(0).to(torch.int32)
        s["live"] = torch.tensor(live, dtype=torch.long, device="cuda")
        s["tok_seq"], s["tok_slot"] = (torch.tensor([t[k] for t in tok], dtype=torch.long, device="cuda")
                                       for k in (0, 1))
        # positions run ahead of the slots where slots were evicted before; an image's
        # tokens share a time and stand in rows and columns
        ahead = torch.randint(0, 5000, (n,), generator=gen, device="cuda")
        pos = torch.zeros((axes, rows), dtype=torch.long, device="cuda")
        pos[:, s["live"]] = ahead[s["tok_seq"]] + s["tok_slot"]
        if axes > 1:
            pos[1, s["live"]] += s["tok_slot"] // 28 % 28
            pos[-1, s["live"]] += s["tok_slot"] % 28
        s["token_positions"] = pos.to(torch.int32)
        s["pair_axis"] = None
        if axes > 1:  # a run of pairs for each axis
            s["pair_axis"] = torch.tensor([min(axes - 1, i * axes // (R // 2)) for i in range(R // 2)],
                                          dtype=torch.uint8, device="cuda")
    return s


# --------------------------------------------------------------- plain form --
def _rotate(x, cos, sin, rotary, interleaved):
    """In the type of cos and sin."""
    x, rest = x[..., :rotary].to(cos.dtype), x[..., rotary:]
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
    P, R = c["page"], c["rotary"]
    pos = s["token_positions"][:, live].double()
    of = pos.t() if s["pair_axis"] is None else pos.t()[:, s["pair_axis"].long()]
    angle = of * s["inv_freq"].double()  # far positions: 64 bits
    cos, sin = angle.cos(), angle.sin()
    s["q_out"][live] = _rotate(s["q"][live], cos.float(), sin.float(), R, c["interleaved"])
    k = _rotate(s["k"][live], cos, sin, R, c["interleaved"])  # quantised: values next to a border
    kc, vc, ks, vs = _parts(s["pool"], s["dim"], s["dtype"])
    page = s["table"][s["tok_seq"], s["tok_slot"] // P].long()
    block, slot = s["tok_slot"] % P // 16, s["tok_slot"] % 16
    kc[page, :, block, :, slot], ks[page, :, block, :, slot] = _quantised(k)
    vc[page, :, block, :, slot], vs[page, :, block, :, slot] = _quantised(s["v"][live])
    if s["weights"] is not None:
        s["weights"][s["tok_seq"], :, s["tok_slot"]] = 0
        s["positions"][s["tok_seq"], :, s["tok_slot"]] = s["token_positions"][0, live][:, None]
    return s["q_out"]


def _attend_plain(s, q):
    c, n, K = s["case"], s["case"]["n_seq"], s["case"]["kv_heads"]
    kc, vc, ks, vs = _parts(s["pool"][s["table"].long()].transpose(1, 2), s["dim"], s["dtype"])
    qg = (q.float() * s["scale"]).view(n, K, c["heads"] // K, -1)
    score = qg @ _values(kc, ks).flatten(2, 4).transpose(-1, -2)
    there = torch.arange(score.shape[-1], device=q.device) < s["seq_len"][:, None]
    score = score.masked_fill(~there[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    w = torch.exp(score - top)
    total = w.sum(-1, keepdim=True)
    w = w / torch.where(total > 0, total, 1.0)
    out = (w @ _values(vc, vs).flatten(2, 4)).flatten(1, 2).to(q.dtype)
    got = dict(out=out, lse=(top + total.log()).flatten(1))
    if s["weights"] is not None:
        s["weights"] += w.sum(2)
        got.update(weights=s["weights"], positions=s["positions"])
    return got


def _expand_plain(s):
    P = s["case"]["page"]
    kc, vc, ks, vs = _parts(s["pool"], s["dim"], s["dtype"])
    at = (s["table"][s["row_seq"], s["row_slot"] // P].long(), slice(None), s["row_slot"] % P // 16, slice(None),
          s["row_slot"] % 16)
    return dict(k=_values(kc[at][..., None, :], ks[at][..., None, :])[:, :, 0].to(s["dtype"]),
                v=_values(vc[at][..., None, :], vs[at][..., None, :])[:, :, 0].to(s["dtype"]))


def _evict_plain(s):
    c, P, keep = s["case"], s["case"]["page"], s["keep"]
    s["both"].copy_(s["before"])  # another step's: what was evicted last time is there again
    weights, positions, lens = s["weights"], s["positions"], s["seq_len"][:, None, None]
    slot = torch.arange(weights.shape[-1], device=weights.device)
    there = slot < lens
    newest = torch.where(there, positions, -1 << 31).amax(-1, keepdim=True).long()
    guarded = there & ((positions < s["first"]) | (positions.long() > newest - s["recent"]))
    order = torch.where(there, weights, -math.inf).sort(dim=-1, descending=True, stable=True).indices
    grade = torch.where(guarded, 0, torch.where(there, 1, 2)).gather(-1, order)
    order = order.gather(-1, grade.sort(dim=-1, stable=True).indices)
    kept = torch.zeros_like(there).expand_as(weights).scatter(-1, order[..., :keep], True) & there
    over = lens > keep
    hole = (over & ~kept & (slot < keep)).nonzero(as_tuple=True)  # row by row, as many as
    come = (over & kept & (slot >= keep)).nonzero(as_tuple=True)  # come from behind
    for part in _parts(s["pool"], s["dim"], s["dtype"]):
        src, dst = ((s["table"][seq, at // P].long(), head, at % P // 16, slice(None), at % 16)
                    for seq, head, at in (come, hole))
        part[dst] = part[src]
    weights[hole] = weights[come]
    positions[hole] = positions[come]
    return dict(length=s["seq_len"].clamp(max=keep), weights=weights, positions=positions, **_expand_plain(s))


def _run_plain(s):
    if s["op"] == "step":
        q = _append_plain(s)
        return dict(q=q, **_attend_plain(s, q))
    if s["op"] == "attend":
        return _attend_plain(s, s["q"])
    if s["op"] == "chunk":
        return dict(q=_append_plain(s), **_expand_plain(s))
    return _evict_plain(s)


# ------------------------------------------------------ the framework's calls --
def _run_own(s):
    from qweninferenceengine_b200 import ops

    op = s["op"]
    kv = ops.PagedKVQ4(s["pool"], s["table"], s["dtype"], weights=s["weights"], positions=s["positions"])
    got, q = {}, s.get("q")
    if op in ("step", "chunk"):
        q = got["q"] = ops.rope_append_paged_q4(
            kv, s["q"], s["k"], s["v"], s["seq_len"], s["inv_freq"], cu_tokens=s["cu_tokens"],
            positions=s["token_positions"], pair_axis=s["pair_axis"],
            interleaved=s["case"]["interleaved"], out=s["q_out"])
    if op in ("step", "attend"):
        got["out"], got["lse"] = ops.attention_paged_q4(kv, q, s["seq_len"], scale=s["scale"], return_lse=True)
        if s["weights"] is not None:
            got.update(weights=s["weights"], positions=s["positions"])
        return got
    lens = s["seq_len"]
    if op == "evict":
        s["both"].copy_(s["before"])  # another step's: what was evicted last time is there again
        lens = ops.evict_paged_q4(kv, lens, s["keep"], n_first=s["first"], n_recent=s["recent"])
        got.update(length=lens, weights=s["weights"], positions=s["positions"])
    got["k"], got["v"] = ops.expand_paged_q4(kv, lens, s["cu"], s["rows"])
    return got


def run(state):
    if own:
        return _run_own(state)
    return _run_plain(state)


# ------------------------------------------------------------------- work ----
def work(case):
    c = case
    n, H, K, D, P = c["n_seq"], c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    lens, new = _lengths(c)
    row = 1.25 * D * K  # of the cache: codes, steps and lows of keys and values
    held, tokens = sum(lens), sum(new)
    table = 4.0 * sum(_pages(x, P) for x in lens) + 4 * n
    rotated = dict(bytes=0.0, flops=0.0)
    if tokens:  # q, k, v read, q written; angles
        rotated = dict(bytes=2.0 * tokens * (2 * H + 2 * K) * D + tokens * (row + 4 * c["axes"]) + 2 * c["rotary"],
                       flops=3.0 * tokens * (H + K) * c["rotary"] + 6.0 * tokens * 2 * K * D)
    if c["op"] in ("step", "attend"):
        weighed = 8.0 * held * K if c["weigh"] else 0.0
        return dict(bytes=rotated["bytes"] - tokens * row + held * row + weighed + table
                    + 2.0 * 2 * n * H * D + 4 * n * H,
                    flops=rotated["flops"] + 4.0 * held * H * D)
    if c["op"] == "chunk":  # every row read back once, the new ones from what was written
        return dict(bytes=rotated["bytes"] + table + held * (row + 4.0 * K * D),
                    flops=rotated["flops"] + 4.0 * held * K * D)
    left = sum(min(x, c["keep"]) for x in lens)
    over = [x for x in lens if x > c["keep"]]
    moved = sum(min(c["keep"], x - c["keep"]) * (c["keep"] / x) for x in over)  # about
    return dict(bytes=8.0 * K * sum(over) + moved * (2 * row + 16 * K) + left * (row + 4.0 * K * D) + table,
                flops=4.0 * left * K * D + 2.0 * K * sum(over))


# ------------------------------------------- the definition, in 64 bits -------
def _exact_groups(x):
    """Codes (as 64-bit numbers), steps and lows of the groups of rows in the cache's type."""
    g = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    low, high = g.min(-1).values.double(), g.max(-1).values.double()
    step = (high.sub(low).div(15)).to(x.dtype).double()
    safe = torch.where(step > 0, step, 1.0)
    code = torch.round((g.double() - low[..., None]) / safe[..., None])
    return torch.where(step[..., None] > 0, code.clamp(0, 15), 0.0), step, low


def _exact_row(s, i, slots):
    """Keys and values [slots, kv_heads, d] of sequence i, in 64 bits."""
    c = s["case"]
    D, P, K = c["head_dim"], c["page"], c["kv_heads"]
    pages = s["pool"][s["table"][i, slots // P].long(), :, slots % P // 16]  # [slots, K, 20 D]
    r = slots % 16
    got = []
    for half in (0, 1):
        groups = []
        for g in range(D // 32):
            at = half * 8 * D + g * 256 + 16 * r
            b = torch.gather(pages, 2, (at[:, None] + torch.arange(16, device="cuda"))[:, None].expand(-1, K, -1))
            at = (16 + 2 * half) * D + g * 64 + 4 * r
            p = torch.gather(pages, 2, (at[:, None] + torch.arange(4, device="cuda"))[:, None].expand(-1, K, -1))
            p = p.contiguous().view(s["dtype"]).double()
            code = torch.empty((*b.shape[:2], 32), dtype=torch.float64, device="cuda")
            code[..., 0::2], code[..., 1::2] = (b % 16).double(), (b // 16).double()
            groups.append(p[..., 1:] + code * p[..., :1])
        got.append(torch.cat(groups, -1))
    return got


def _exact_append(s):
    """(q, rows that the appended tokens stand for: keys and values in 64 bits)."""
    c, live = s["case"], s["live"]
    R, half = c["rotary"], c["rotary"] // 2
    which = torch.zeros(half, dtype=torch.long, device="cuda") if s["pair_axis"] is None else s["pair_axis"].long()
    angle = s["token_positions"].double()[which][:, live].t() * s["inv_freq"].double()
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]

    def spun(x):
        x = x[live].double()
        if c["interleaved"]:
            z = torch.view_as_complex(x[..., :R].reshape(*x.shape[:-1], half, 2).contiguous()) * turn
            x[..., :R] = torch.view_as_real(z).reshape(*x.shape[:-1], R)
        else:
            z = torch.complex(x[..., :half].contiguous(), x[..., half:R].contiguous()) * turn
            x[..., :half], x[..., half:R] = z.real, z.imag
        return x

    q = s["q_out"].double()
    q[live] = spun(s["q"])
    rows = []
    for x in (spun(s["k"]).to(s["dtype"]), s["v"][live]):
        code, step, low = _exact_groups(x)
        rows.append((low[..., None] + code * step[..., None]).flatten(-2))
    return q, rows


def exact(case, seed):
    s = prepare(case, seed)
    c, K, P = case, case["kv_heads"], case["page"]
    lens, _ = _lengths(c)
    got, new_rows = {}, None
    if c["op"] in ("step", "chunk"):
        got["q"], new_rows = _exact_append(s)
    if c["op"] == "evict":
        return _exact_evict(s, lens)
    if c["op"] == "chunk":
        ks, vs = [], []
        for i, x in enumerate(lens):
            k, v = _exact_row(s, i, torch.arange(x, device="cuda"))
            mine = s["tok_seq"] == i
            k[s["tok_slot"][mine]], v[s["tok_slot"][mine]] = new_rows[0][mine], new_rows[1][mine]
            ks.append(k)
            vs.append(v)
        return dict(k=torch.cat(ks), v=torch.cat(vs), **got)
    outs, lses = [], []
    weights = s["weights"].double() if c["weigh"] else None
    q = s["q"].double()
    if c["op"] == "step":
        q = got["q"].to(s["dtype"]).double()  # the attention takes what was rounded
        if c["weigh"]:
            weights[s["tok_seq"], :, s["tok_slot"]] = 0.0
            s["positions"][s["tok_seq"], :, s["tok_slot"]] = s["token_positions"][0, s["live"]][:, None]
    G = c["heads"] // K
    for i, x in enumerate(lens):
        k, v = _exact_row(s, i, torch.arange(x, device="cuda"))
        if new_rows is not None and x:
            at = (s["tok_seq"] == i).nonzero()[0, 0]
            k[x - 1], v[x - 1] = new_rows[0][at], new_rows[1][at]
        out, lse = [], []
        for h in range(K):
            z = q[i, h * G:(h + 1) * G] @ k[:, h].T * s["scale"]
            if x:
                w = torch.softmax(z, -1)
                out.append(w @ v[:, h])
                lse.append(torch.logsumexp(z, -1))
                if weights is not None:
                    weights[i, h, :x] += w.sum(0)
            else:
                out.append(torch.zeros_like(q[i, :G]))
                lse.append(torch.full((G,), -math.inf, dtype=torch.float64, device="cuda"))
        outs.append(torch.cat(out))
        lses.append(torch.cat(lse))
    got.update(out=torch.stack(outs), lse=torch.stack(lses))
    if weights is not None:
        got.update(weights=weights, positions=s["positions"])
    return got


def _exact_evict(s, lens):
    c, keep, K = s["case"], s["keep"], s["case"]["kv_heads"]
    weights, positions = s["weights"].clone(), s["positions"].clone()
    ks, vs = [], []
    for i, x in enumerate(lens):
        k, v = _exact_row(s, i, torch.arange(x, device="cuda"))
        if x > keep:
            w, p = s["weights"][i, :, :x].tolist(), s["positions"][i, :, :x].tolist()
            for h in range(K):
                newest = max(p[h])
                rank = sorted(range(x), key=lambda j: (
                    not (p[h][j] < s["first"] or p[h][j] > newest - s["recent"]), -w[h][j], j))
                kept = set(rank[:keep])
                dst = torch.tensor([j for j in range(keep) if j not in kept], dtype=torch.long, device="cuda")
                src = torch.tensor([j for j in range(keep, x) if j in kept], dtype=torch.long, device="cuda")
                for t in (k[:, h], v[:, h], weights[i, h], positions[i, h]):
                    t[dst] = t[src]
        ks.append(k[:keep])
        vs.append(v[:keep])
    return dict(length=torch.tensor([min(x, keep) for x in lens], dtype=torch.int32, device="cuda"),
                weights=weights.double(), positions=positions, k=torch.cat(ks), v=torch.cat(vs))
