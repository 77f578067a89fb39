"""The attention half of a layer that streams its experts, as cases that can be timed and compared.

What a decode step does beside the routed blocks: the new tokens get their place in a paged cache (plan), their queries and
keys are rotated by their positions (rotate), keys and values go to the cache as 4-bit values (store), and each request's
queries attend to its pages (cached). A prompt, and a training step, attend to keys and values of 16 bits (attend). The cache
shares HBM with the experts: at 4 bits it leaves the slots nearly three quarters of what it would take at 16.

Every case is a dict of plain values; "op" names the operator:

  rotate   pairs of a head's values turned by position x frequency ("grad": the gradients too)
  plan     pages, positions and slots of a step's tokens from the requests' lengths
  store    keys and values to their slots as 4-bit values, and back
  cached   softmax(q K^T scale) V over the pages of each request
  attend   softmax(q K^T scale) V over packed sequences ("grad": dq, dk, dv too)

`own` chooses who computes: False, elementary torch operations in 32 bits (angles in 64); True, the library.

The cache, as both forms read it. A page holds 64 tokens; for each head that keeps keys and values, 72 head_dim bytes:
  keys          [64 tokens][4 g][head_dim / 32 blocks b][4 bytes]
  key scales    [64 tokens][blocks] half precision
  value scales  [64 tokens][blocks] half precision
  values        [blocks][64 tokens][16 bytes]
Byte j of a block's 16 has value j in its low and value 16 + j in its high four bits, each plus 8 (a key's byte 4 g + i stands
at [g][b][i]); a block's values are these whole numbers, -8 to 7, times its scale.
"""
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
PAGE, BLOCK = 64, 32


def listed():
    return [
        # One token of a decode step: its queries and keys, all latency.
        {"name": "rotate-token", "op": "rotate", "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128, "rotated": 128, "interleaved": False,
         "factor": 1.0, "trained": 0, "far": 32768, "type": "bf16", "grad": False},
        # A training step, half of each head rotated, interleaved pairs, frequencies blended for four times the trained length.
        {"name": "rotate-train", "op": "rotate", "tokens": 8191, "heads": 32, "kv_heads": 4, "dim": 128, "rotated": 64, "interleaved": True,
         "factor": 4.0, "trained": 8192, "far": 32768, "type": "bf16", "grad": True},
        # A decode step of 32 requests: a page for one in 64 of them.
        {"name": "plan-step", "op": "plan", "requests": 32, "longest": 32768, "rows": 32, "mix": False},
        # A step that admits prompts and drops finished requests among 2,000 that go on.
        {"name": "plan-admit", "op": "plan", "requests": 2047, "longest": 32768, "rows": 65536, "mix": True},
        # The keys and values of a decode step.
        {"name": "store-step", "op": "store", "tokens": 32, "kv_heads": 8, "dim": 128, "type": "bf16"},
        # The keys and values of a prompt of odd length.
        {"name": "store-prompt", "op": "store", "tokens": 8191, "kv_heads": 8, "dim": 128, "type": "f16"},
        # One request's token behind 4,096 others: few rows, the cache split over the chip.
        {"name": "cached-token", "op": "cached", "requests": 1, "longest": 4097, "fresh": 1, "kv_heads": 8, "group": 4, "dim": 128,
         "type": "bf16"},
        # A batch of ragged lengths, eight query heads to each kept one.
        {"name": "cached-batch", "op": "cached", "requests": 64, "longest": 8191, "fresh": 1, "kv_heads": 4, "group": 8, "dim": 128,
         "type": "bf16"},
        # Four long requests, half precision, three tokens each (two of them drafted): 370 MB of cache.
        {"name": "cached-long", "op": "cached", "requests": 4, "longest": 131071, "fresh": 3, "kv_heads": 8, "group": 4, "dim": 128,
         "type": "f16"},
        # One prompt of odd length: the largest products.
        {"name": "attend-prompt", "op": "attend", "tokens": 8191, "sequences": 1, "prefix": 0, "kv_heads": 8, "group": 4, "dim": 128,
         "causal": True, "type": "bf16", "grad": False},
        # A small ragged training step in half precision.
        {"name": "attend-train-small", "op": "attend", "tokens": 301, "sequences": 3, "prefix": 0, "kv_heads": 2, "group": 2, "dim": 64,
         "causal": True, "type": "f16", "grad": True},
        # A training step over packed sequences: every gradient.
        {"name": "attend-train", "op": "attend", "tokens": 8192, "sequences": 3, "prefix": 0, "kv_heads": 8, "group": 4, "dim": 128,
         "causal": True, "type": "bf16", "grad": True},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["rotate", "rotate", "plan", "plan", "store", "cached", "cached", "cached", "attend", "attend", "attend"])
    kind = rng.choice(["bf16", "bf16", "f16"])
    if op == "rotate":
        dim = rng.choice([64, 80, 96, 128, 128])
        return {"op": op, "tokens": _spread(rng, 1, 8192), "heads": _spread(rng, 1, 32), "kv_heads": _spread(rng, 1, 8), "dim": dim,
                "rotated": rng.choice([dim, dim, dim // 2]), "interleaved": rng.random() < 0.5, "factor": rng.choice([1.0, 1.0, 8.0, 2.5]),
                "trained": rng.choice([0, 4096, 8192]), "far": rng.choice([512, 32768, 1 << 20]),
                "type": rng.choice(["bf16", "f16", "f32"]), "grad": rng.random() < 0.5}
    if op == "plan":
        mix, requests = rng.random() < 0.6, _spread(rng, 1, 2047)
        return {"op": op, "requests": requests, "longest": _spread(rng, 64, 32768), "mix": mix,
                "rows": requests + (_spread(rng, 1, 32768) if mix else rng.choice([0, 0, 7]))}
    if op == "store":
        return {"op": op, "tokens": _spread(rng, 1, 8192), "kv_heads": _spread(rng, 1, 8), "dim": rng.choice([32, 64, 96, 128, 128]), "type": kind}
    if op == "cached":
        case = {"op": op, "requests": _spread(rng, 1, 128), "longest": _spread(rng, 8, 131071), "fresh": rng.choice([1, 1, 1, 2, 5, 8]),
                "kv_heads": _spread(rng, 1, 8), "group": rng.choice([1, 2, 4, 5, 8, 16]), "dim": rng.choice([32, 64, 96, 128, 128]), "type": kind}
        while case["requests"] > 1 and case["requests"] * case["longest"] * case["kv_heads"] * case["group"] * case["dim"] > 1e9:
            case["requests"] -= 1
        return case
    case = {"op": op, "tokens": _spread(rng, 1, 8192), "sequences": _spread(rng, 1, 8), "prefix": rng.choice([0, 0, 0, 77, 512]),
            "kv_heads": _spread(rng, 1, 8), "group": rng.choice([1, 2, 4, 4]), "dim": rng.choice([32, 64, 72, 128, 128]),
            "causal": rng.random() < 0.8, "type": kind, "grad": rng.random() < 0.5}
    case["sequences"] = min(case["sequences"], case["tokens"])
    while work(case)["flops"] > work(listed()[-1])["flops"] / 2:
        case["tokens"] -= 64
    return case


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, kind, sigma=1.0):
    return (torch.randn(shape, device="cuda", generator=g) * sigma).to(TYPES[kind])


def _ragged(total, n):
    """n lengths, unlike each other, of this sum; each 1 at least."""
    rng = random.Random(total * 31 + n)
    share = [rng.uniform(0.3, 1.7) for _ in range(n)]
    at = [0] + [round((total - n) * sum(share[:i + 1]) / sum(share)) for i in range(n)]
    return [b - a + 1 for a, b in zip(at, at[1:])]


def _ends(case):
    """The lengths of a cached case's requests, the longest first."""
    rng = random.Random(case["requests"] * 131 + case["longest"])
    low = max(case["fresh"], case["longest"] // 8)
    return [max(case["longest"], case["fresh"])] + [rng.randint(low, max(low, case["longest"])) for _ in range(case["requests"] - 1)]


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _first(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return _i32(at)


def _quantized(x):
    """(whole numbers 0..15, scales in half precision) of rows of blocks: the value of the largest size (of equal ones the
    lowest) over -8 is the scale, rounded to half precision; the others are rounded to whole steps of it."""
    b = x.float().reshape(*x.shape[:-1], -1, BLOCK)
    size = b.abs()
    at = (size == size.amax(-1, keepdim=True)).int().cumsum(-1).eq(0).sum(-1, keepdim=True)  # ties: the lowest
    scale = (torch.gather(b, -1, at) / -8).half()
    steps = torch.where(scale == 0, 0.0, b / scale.float())
    return (torch.round(steps) + 8).clamp(0, 15).to(torch.uint8), scale[..., 0]


def _pages(k, v):
    """Pages [n][heads][72 dim] of keys and values [n x 64][heads][dim]."""
    (rows, heads, dim), out = k.shape, []
    n, nb = rows // PAGE, dim // BLOCK
    for x in (k, v):
        q, s = _quantized(x)
        q = (q[..., :16] | q[..., 16:] << 4).view(n, PAGE, heads, nb, 16).transpose(1, 2)  # [n][heads][64][nb][16]
        out.append((q, s.view(n, PAGE, heads, nb).transpose(1, 2).contiguous().view(torch.uint8).reshape(n, heads, -1)))
    (kq, ks), (vq, vs) = out
    kq = kq.reshape(n, heads, PAGE, nb, 4, 4).transpose(3, 4).reshape(n, heads, -1)
    vq = vq.transpose(2, 3).reshape(n, heads, -1)
    return torch.cat([kq, ks, vs, vq], 2).contiguous()


def _prepare_plan(s, case, seed):
    rng, n, longest = random.Random(seed), case["requests"], case["longest"]
    lengths, fresh, left = [], [], case["rows"]
    for i in range(n):
        u = rng.random()
        lengths.append(_spread(rng, 1, longest))
        fresh.append(1)
        if case["mix"] and u < 0.1:
            fresh[i] = -1  # the request has ended
        elif case["mix"] and u < 0.15:
            fresh[i] = 0
        elif case["mix"] and u < 0.4:
            lengths[i], fresh[i] = 0, _spread(rng, 1, longest)  # a prompt
        fresh[i] = min(fresh[i], max(0, left - (n - 1 - i)))
        left -= max(fresh[i], 0)
    width = longest // PAGE + 2
    pages = [(a + PAGE - 1) // PAGE for a in lengths]
    order = torch.randperm(n * width, generator=torch.Generator().manual_seed(seed)).to(torch.int32)  # a pool that holds every table
    table, at = torch.full((n, width), -1, dtype=torch.int32), n * width
    for i, p in enumerate(pages):
        table[i, :p] = order[at - p:at]
        at -= p
    order[at:] = -1
    s.update(lengths=_i32(lengths), fresh=_i32(fresh), table=table.cuda(), free=order.cuda(), n_free=_i32([at]))


def prepare(case, seed):
    g, s = _generator(seed), dict(case)
    op = case["op"]
    if op == "rotate":
        for name, heads in (("q", case["heads"]), ("k", case["kv_heads"])):
            s[name] = _normal(g, (case["tokens"], heads, case["dim"]), case["type"])
            if case["grad"]:
                s["d" + name] = _normal(g, (case["tokens"], heads, case["dim"]), case["type"])
        s["positions"] = torch.randint(0, case["far"], (case["tokens"],), device="cuda", generator=g, dtype=torch.int32)
        s["amplitude"] = 1.0 if case["factor"] == 1 else 0.1 * math.log(case["factor"]) + 1
        if own:
            s["plan"] = _rotary(s)
    elif op == "plan":
        _prepare_plan(s, case, seed)
    elif op == "store":
        t, pages = case["tokens"], case["tokens"] // PAGE + 4
        s["k"], s["v"] = (_normal(g, (t, case["kv_heads"], case["dim"]), case["type"], sigma) for sigma in (2.0, 0.7))
        # pages in no order, the tokens inside them one after the other, from the middle of the first one on
        order = torch.randperm(pages, device="cuda", generator=g)
        at = torch.arange(t, device="cuda") + 13
        s["slots"] = (order[at // PAGE] * PAGE + at % PAGE).to(torch.int32)
        s["pages"] = torch.zeros((pages, case["kv_heads"], 72 * case["dim"]), dtype=torch.uint8, device="cuda")
    elif op == "cached":
        ends, kv, dim = _ends(case), case["kv_heads"], case["dim"]
        need = [(e + PAGE - 1) // PAGE for e in ends]
        n, width = sum(need) + 3, max(need)
        order, table = torch.randperm(n, device="cuda", generator=g).to(torch.int32), torch.full((len(ends), width), -1, dtype=torch.int32, device="cuda")
        at = 0
        for i, p in enumerate(need):
            table[i, :p] = order[at:at + p]
            at += p
        s["pages"] = torch.empty((n, kv, 72 * dim), dtype=torch.uint8, device="cuda")
        for p in range(0, n, 512):
            rows = min(512, n - p) * PAGE
            s["pages"][p:p + 512] = _pages(_normal(g, (rows, kv, dim), "f16", 1.0), _normal(g, (rows, kv, dim), "f16", 0.5))
        s["q"] = _normal(g, (len(ends) * case["fresh"], kv * case["group"], dim), case["type"])
        s["table"], s["ends"], s["first"] = table, _i32(ends), _first([case["fresh"]] * len(ends))
        if own:
            from tierstream_amd import attn
            s["cache"] = attn.Cache(s["pages"], kv, dim)
    else:
        kv, dim = case["kv_heads"], case["dim"]
        s["lengths"] = _ragged(case["tokens"], case["sequences"])
        s["k_lengths"] = [n + case["prefix"] for n in s["lengths"]]
        s["first"], s["k_first"] = _first(s["lengths"]), _first(s["k_lengths"])
        s["q"] = _normal(g, (case["tokens"], kv * case["group"], dim), case["type"])
        s["k"], s["v"] = (_normal(g, (sum(s["k_lengths"]), kv, dim), case["type"]) for _ in range(2))
        if case["grad"]:
            s["dout"] = _normal(g, s["q"].shape, case["type"], 0.05)
    return s


# ---- the plain form -------------------------------------------------------------------------------------------------
def _frequencies(s):
    """Radians a position of each pair: base^(-2 i / rotated), divided by factor where the trained length holds fewer than one
    turn, left where it holds more than four, blended between."""
    f = 10000.0 ** (-torch.arange(0, s["rotated"], 2, dtype=torch.float64, device="cuda") / s["rotated"])
    if s["factor"] == 1:
        return f
    keep = ((s["trained"] * f / (2 * math.pi) - 1) / (4 - 1)).clamp(0, 1)
    return f * (keep + (1 - keep) / s["factor"])


def _turned(x, cos, sin, s):
    r, wide = s["rotated"], x.float()
    part = wide[..., :r]
    a, b = (part[..., 0::2], part[..., 1::2]) if s["interleaved"] else (part[..., :r // 2], part[..., r // 2:])
    new = (a * cos - b * sin, a * sin + b * cos)
    part = torch.stack(new, -1).flatten(-2) if s["interleaved"] else torch.cat(new, -1)
    return torch.cat([part, wide[..., r:]], -1).to(x.dtype)


def _plain_rotate(s):
    angle = s["positions"].double()[:, None] * _frequencies(s)
    cos, sin = ((t * s["amplitude"]).float()[:, None] for t in (torch.cos(angle), torch.sin(angle)))
    out = {"q": _turned(s["q"], cos, sin, s), "k": _turned(s["k"], cos, sin, s)}
    if s["grad"]:
        out.update(dq=_turned(s["dq"], cos, -sin, s), dk=_turned(s["dk"], cos, -sin, s))
    return out


def _flat(counts):
    """(owner, number inside it) of each of sum(counts) things."""
    owner = torch.repeat_interleave(torch.arange(len(counts), device="cuda"), counts)
    return owner, torch.arange(len(owner), device="cuda") - (counts.cumsum(0) - counts)[owner]


def _plain_plan(s):
    lengths, fresh, table, free = s["lengths"].long(), s["fresh"].long(), s["table"], s["free"]
    add, over = fresh.clamp_min(0), fresh < 0
    have = (lengths + PAGE - 1) // PAGE
    ends = torch.where(over, 0, lengths + add)
    need = torch.where(over, 0, (ends + PAGE - 1) // PAGE - have)
    owner, j = _flat(torch.where(over, have, 0))
    count = s["n_free"].long() + len(owner)
    free[s["n_free"].long() + torch.arange(len(owner), device="cuda")] = table[owner, j]
    owner, j = _flat(need)
    table[owner, have[owner] + j] = free[count - 1 - torch.arange(len(owner), device="cuda")]
    owner, j = _flat(add)
    positions, slots = (torch.full((s["rows"],), -1, dtype=torch.int32, device="cuda") for _ in range(2))
    at = lengths[owner] + j
    positions[:len(owner)] = at.int()
    slots[:len(owner)] = table[owner, at // PAGE] * PAGE + (at % PAGE).int()
    first = torch.zeros(len(add) + 1, dtype=torch.int32, device="cuda")
    first[1:] = add.cumsum(0)
    return {"ends": ends.int(), "left": (count - need.sum()).int(), "table": table, "free": free, "first": first, "positions": positions,
            "slots": slots, "status": torch.zeros(1, dtype=torch.int32, device="cuda")}


def _parts(pages, dim):
    """(key bytes, key scales, value scales, value bytes) of pages, each [..., 64][blocks] with 16 bytes or one scale."""
    kq, ks, vs, vq = pages.split([32 * dim, 4 * dim, 4 * dim, 32 * dim], -1)
    lead, nb = pages.shape[:-1], dim // BLOCK
    kq = kq.reshape(*lead, PAGE, 4, nb, 4).transpose(-3, -2).reshape(*lead, PAGE, nb, 16)
    vq = vq.reshape(*lead, nb, PAGE, 16).transpose(-3, -2)
    ks, vs = (t.contiguous().view(torch.float16).view(*lead, PAGE, nb) for t in (ks, vs))
    return kq, ks, vs, vq


def _numbers(q, s):
    return ((torch.cat([q & 15, q >> 4], -1).float() - 8) * s.float()[..., None]).flatten(-2)


def _plain_store(s):
    pages, at, heads, dim = s["pages"], s["slots"].long(), s["kv_heads"], s["dim"]
    page, row, nb = at // PAGE, at % PAGE, dim // BLOCK
    out = []
    for name, begin, scale_at in (("k", 0, 32 * dim), ("v", 40 * dim, 36 * dim)):
        q, scale = _quantized(s[name])
        q = q[..., :16] | q[..., 16:] << 4  # [tokens][heads][nb][16]
        scales = pages[:, :, scale_at:scale_at + 4 * dim].view(len(pages), heads, PAGE, 2 * nb)
        scales[page, :, row] = scale.contiguous().view(torch.uint8)
        room = pages[:, :, begin:begin + 32 * dim]
        if name == "k":
            room = room.view(len(pages), heads, PAGE, 4, nb, 4)
            room[page, :, row] = q.view(len(at), heads, nb, 4, 4).transpose(2, 3)
            back = room[page, :, row].transpose(2, 3).reshape(len(at), heads, nb, 16)
        else:
            room = room.view(len(pages), heads, nb, PAGE, 16)
            room[page, :, :, row] = q
            back = room[page, :, :, row]
        out.append(_numbers(back, scales[page, :, row].contiguous().view(torch.float16)).to(s[name].dtype))
    return {"k": out[0], "v": out[1]}


def _plain_cached(s):
    n, f, kv, group, dim = s["requests"], s["fresh"], s["kv_heads"], s["group"], s["dim"]
    kq, ks, vs, vq = _parts(s["pages"][s["table"].clamp_min(0).long()], dim)  # [n][width][kv][64]...
    k, v = (_numbers(q, t).permute(0, 2, 1, 3, 4).reshape(n * kv, -1, dim) for q, t in ((kq, ks), (vq, vs)))
    q = s["q"].float().view(n, f, kv, group, dim).permute(0, 2, 1, 3, 4).reshape(n * kv, f * group, dim)
    scores = (q @ k.transpose(1, 2)).view(n, kv, f, group, -1) * dim ** -0.5
    last = s["ends"][:, None] - f + torch.arange(f, device="cuda")  # [n][f]: the last key each token attends to
    seen = torch.arange(scores.shape[-1], device="cuda") <= last[:, :, None]
    scores = scores.masked_fill(~seen[:, None, :, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    v = v.masked_fill(~(torch.arange(v.shape[1], device="cuda") < s["ends"][:, None]).repeat_interleave(kv, 0)[..., None], 0.0)
    out = (p.view(n * kv, f * group, -1) @ v).view(n, kv, f, group, dim).permute(0, 2, 1, 3, 4)
    return {"out": out.reshape(n * f, kv * group, dim).to(s["q"].dtype)}


def _plain_attend(s):
    group, scale, kind = s["group"], s["dim"] ** -0.5, s["q"].dtype
    out = {"out": torch.empty_like(s["q"]), "lse": torch.empty((s["q"].shape[1], s["tokens"]), device="cuda")}
    if s["grad"]:
        out.update(dq=torch.empty_like(s["q"]), dk=torch.empty_like(s["k"]), dv=torch.empty_like(s["v"]))
    a = b = 0
    for n, m in zip(s["lengths"], s["k_lengths"]):
        q = s["q"][a:a + n].float().transpose(0, 1)
        k, v = (s[x][b:b + m].float().transpose(0, 1).repeat_interleave(group, 0) for x in ("k", "v"))
        scores = q @ k.transpose(1, 2) * scale
        if s["causal"]:
            ahead = torch.arange(m, device="cuda") > torch.arange(n, device="cuda")[:, None] + (m - n)
            scores = scores.masked_fill(ahead, -math.inf)
        top = scores.amax(-1, keepdim=True)
        p = torch.exp(scores - top)
        total = p.sum(-1, keepdim=True)
        out["lse"][:, a:a + n] = (top + torch.log(total))[..., 0]
        p = p / total
        o = p @ v
        out["out"][a:a + n] = o.transpose(0, 1).to(kind)
        if s["grad"]:
            do = s["dout"][a:a + n].float().transpose(0, 1)
            dv = (p.transpose(1, 2) @ do).view(-1, group, m, s["dim"]).sum(1)
            ds = p * (do @ v.transpose(1, 2) - (do * o).sum(-1, keepdim=True))
            dk = (ds.transpose(1, 2) @ q).view(-1, group, m, s["dim"]).sum(1) * scale
            out["dq"][a:a + n] = (ds @ k * scale).transpose(0, 1).to(kind)
            out["dk"][b:b + m], out["dv"][b:b + m] = dk.transpose(0, 1).to(kind), dv.transpose(0, 1).to(kind)
        a, b = a + n, b + m
    return out


# ---- the library's calls --------------------------------------------------------------------------------------------
def _stream():
    return torch.cuda.current_stream().cuda_stream


def _room(n):
    return torch.empty(n, dtype=torch.uint8, device="cuda")


def _rotary(s):
    from tierstream_amd import attn
    return attn.Rotary(s["rotated"], base=10000.0, interleaved=s["interleaved"], factor=s["factor"], trained=s["trained"], low=1.0, high=4.0,
                       amplitude=s["amplitude"])


def _own_rotate(s):
    from tierstream_amd import attn
    out = {"q": torch.empty_like(s["q"]), "k": torch.empty_like(s["k"])}
    attn.rotate(s["plan"], s["positions"], s["q"], s["k"], out["q"], out["k"], stream=_stream())
    if s["grad"]:
        out.update(dq=torch.empty_like(s["q"]), dk=torch.empty_like(s["k"]))
        attn.rotate(s["plan"], s["positions"], s["dq"], s["dk"], out["dq"], out["dk"], backward=True, stream=_stream())
    return out


def _own_plan(s):
    from tierstream_amd import attn
    n, new = s["requests"], lambda size: torch.empty(size, dtype=torch.int32, device="cuda")  # noqa: E731
    out = {"ends": new(n), "left": new(1), "table": s["table"], "free": s["free"], "first": new(n + 1), "positions": new(s["rows"]),
           "slots": new(s["rows"]), "status": new(1)}
    attn.plan(s["lengths"], s["fresh"], s["table"], s["free"], s["n_free"], out["first"], out["positions"], out["slots"], out["status"],
              ends=out["ends"], left=out["left"], stream=_stream())
    return out


def _own_store(s):
    from tierstream_amd import attn
    cache = attn.Cache(s["pages"], s["kv_heads"], s["dim"])
    attn.store(cache, s["k"], s["v"], s["slots"], stream=_stream())
    k, v = torch.empty_like(s["k"]), torch.empty_like(s["v"])
    attn.load(cache, s["slots"], k, v, stream=_stream())
    return {"k": k, "v": v}


def _own_cached(s):
    from tierstream_amd import attn
    out = torch.empty_like(s["q"])
    ws = _room(attn.attend_cached_workspace(s["cache"], s["q"], s["table"]))
    attn.attend_cached(s["cache"], s["q"], out, s["table"], s["ends"], s["first"], workspace=ws, stream=_stream())
    return {"out": out}


def _own_attend(s):
    from tierstream_amd import attn
    q, k, v = s["q"], s["k"], s["v"]
    out = {"out": torch.empty_like(q), "lse": torch.empty((q.shape[1], s["tokens"]), device="cuda")}
    where = {"first": s["first"], "k_first": s["k_first"], "causal": s["causal"], "stream": _stream()}
    attn.attend(q, k, v, out["out"], lse=out["lse"], **where)
    if s["grad"]:
        out.update(dq=torch.empty_like(q), dk=torch.empty_like(k), dv=torch.empty_like(v))
        attn.attend_backward(q, k, v, out["out"], s["dout"], out["lse"], out["dq"], out["dk"], out["dv"],
                             workspace=_room(attn.attend_backward_workspace(q, k)), **where)
    return out


_PLAIN = {"rotate": _plain_rotate, "plan": _plain_plan, "store": _plain_store, "cached": _plain_cached, "attend": _plain_attend}
_OWN = {"rotate": _own_rotate, "plan": _own_plan, "store": _own_store, "cached": _own_cached, "attend": _own_attend}


def run(state):
    return (_OWN if own else _PLAIN)[state["op"]](state)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "rotate":
        wide, heads = 4 if case["type"] == "f32" else 2, case["heads"] + case["kv_heads"]
        n = case["tokens"] * heads * case["dim"] * (2 if case["grad"] else 1)
        return {"bytes": 2 * wide * n + 4 * case["tokens"], "flops": 3 * case["tokens"] * heads * case["rotated"] * (2 if case["grad"] else 1)}
    if op == "plan":
        n, rows = case["requests"], case["rows"]
        return {"bytes": 4 * (4 * n + 2 * rows + rows / PAGE), "flops": 8 * n + 4 * rows}
    if op == "store":
        n = 2 * case["tokens"] * case["kv_heads"] * case["dim"]
        return {"bytes": 2 * n + 2 * n + 2 * n * 18 / 32 + 4 * case["tokens"], "flops": 6 * n}
    if op == "cached":
        f, heads, dim = case["fresh"], case["kv_heads"] * case["group"], case["dim"]
        tokens = sum(_ends(case))
        return {"bytes": tokens * case["kv_heads"] * dim * 9 / 8 + 4 * case["requests"] * f * heads * dim, "flops": 4 * tokens * f * heads * dim}
    lengths, heads, dim = _ragged(case["tokens"], case["sequences"]), case["kv_heads"] * case["group"], case["dim"]
    keys = case["tokens"] + case["sequences"] * case["prefix"]
    pairs = sum(n * case["prefix"] + n * (n + 1) / 2 if case["causal"] else n * (n + case["prefix"]) for n in lengths)
    size = 2 * dim * (2 * case["tokens"] * heads + 2 * keys * case["kv_heads"])
    if case["grad"]:  # out, dout and dq once more, dk and dv
        return {"bytes": size + 2 * dim * (2 * case["tokens"] * heads + 2 * keys * case["kv_heads"]), "flops": 14 * pairs * heads * dim}
    return {"bytes": size, "flops": 4 * pairs * heads * dim}


# ---- in 64 bits, from the definitions -------------------------------------------------------------------------------
def _exact_rotate(s):
    """A pair (a, b) is the complex number a + b i; its position's turn multiplies it."""
    r, turns = s["rotated"], []
    for i in range(r // 2):
        f = math.exp(-math.log(10000.0) * 2 * i / r)
        if s["factor"] != 1:
            inside = s["trained"] / (2 * math.pi / f)  # turns inside the trained length
            keep = min(1.0, max(0.0, (inside - 1.0) / 3.0))
            f = keep * f + (1 - keep) * f / s["factor"]
        turns.append(f)
    angle = torch.outer(s["positions"].double(), torch.tensor(turns, dtype=torch.float64, device="cuda"))[:, None]
    out = {}
    for name, sign in (("q", 1.0), ("k", 1.0), ("dq", -1.0), ("dk", -1.0)):
        if name not in s:
            continue
        y = s[name].double().clone()
        first, second = (slice(0, r, 2), slice(1, r, 2)) if s["interleaved"] else (slice(0, r // 2), slice(r // 2, r))
        z = torch.complex(y[..., first], y[..., second]) * torch.polar(torch.full_like(angle, s["amplitude"]), sign * angle)
        y[..., first], y[..., second] = z.real, z.imag
        out[name] = y
    return out


def _exact_plan(s):
    """Request after request, on the host."""
    lengths, fresh, table = s["lengths"].tolist(), s["fresh"].tolist(), s["table"].cpu().tolist()
    room, count = s["free"].cpu().tolist(), int(s["n_free"][0])
    first, positions, slots, ends = [0], [], [], []
    for i, f in enumerate(fresh):
        if f < 0:
            for j in range(-(-lengths[i] // PAGE)):
                room[count] = table[i][j]
                count += 1
    for i, f in enumerate(fresh):
        ends.append(0 if f < 0 else lengths[i] + f)
        for at in range(lengths[i], ends[i]):
            if at % PAGE:
                page = table[i][at // PAGE]
            else:
                count -= 1
                page = table[i][at // PAGE] = room[count]
            positions.append(at)
            slots.append(page * PAGE + at % PAGE)
        first.append(len(positions))
    rest = [-1] * (s["rows"] - len(positions))
    return {"ends": _i32(ends), "left": _i32([count]), "table": _i32(table), "free": _i32(room), "first": _i32(first),
            "positions": _i32(positions + rest), "slots": _i32(slots + rest), "status": _i32([0])}


def _exact_block(x):
    """What 4 bits a value leave of rows of blocks."""
    b = x.double().unflatten(-1, (-1, BLOCK))
    low, high = b.min(-1, keepdim=True), b.max(-1, keepdim=True)
    big = torch.where(high.values.abs() > low.values.abs(), high.values, low.values)
    tied = high.values == -low.values  # of the two sizes alike, the one that stands first
    plus, minus = (b == high.values).int().argmax(-1, keepdim=True), (b == low.values).int().argmax(-1, keepdim=True)
    big = torch.where(tied & (plus < minus), high.values, torch.where(tied, low.values, big))
    step = (-big / 8).half().double()
    whole = torch.where(step == 0, 0.0, torch.round(b / torch.where(step == 0, 1.0, step))).clamp(-8, 7)
    return (whole * step).flatten(-2)


def _exact_kept(raw, dim):
    """Keys and values [heads][tokens][dim] of pages [n][heads][72 dim]."""
    n, heads, nb = raw.shape[0], raw.shape[1], dim // BLOCK
    keys = raw[..., :32 * dim].view(n, heads, PAGE, 4, nb, 4)
    values = raw[..., 40 * dim:].view(n, heads, nb, PAGE, 16)
    scales = raw[..., 32 * dim:40 * dim].contiguous().view(torch.float16).double().view(n, heads, 2, PAGE, nb)
    out = torch.empty((2, n, heads, PAGE, nb, 32), dtype=torch.float64, device=raw.device)
    for j in range(16):
        for which, byte in ((0, keys[:, :, :, j // 4, :, j % 4]), (1, values[..., j].transpose(2, 3))):
            low = byte % 16
            out[which, ..., j] = low.double() - 8
            out[which, ..., 16 + j] = torch.div(byte, 16, rounding_mode="floor").double() - 8
    for which in range(2):
        out[which] *= scales[:, :, which, :, :, None]
    return out.reshape(2, n, heads, PAGE, dim).transpose(1, 2).reshape(2, heads, n * PAGE, dim)


def _exact_cached(s):
    f, group, dim = s["fresh"], s["group"], s["dim"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, end in enumerate(_ends(s)):
        used = s["table"][i, :(end + PAGE - 1) // PAGE].long()
        for h in range(s["kv_heads"]):
            k, v = _exact_kept(s["pages"][used, h:h + 1], dim)[:, 0, :end]
            for t in range(f):
                upto = end - f + t + 1
                w = torch.softmax(s["q"][i * f + t, h * group:(h + 1) * group].double() @ k[:upto].T / math.sqrt(dim), -1)
                out[i * f + t, h * group:(h + 1) * group] = w @ v[:upto]
    return {"out": out}


def _exact_attend(s):
    group, root = s["group"], math.sqrt(s["dim"])
    new = lambda x: torch.zeros(s[x].shape, dtype=torch.float64, device="cuda")  # noqa: E731
    out = {"out": new("q"), "lse": torch.empty((s["q"].shape[1], s["tokens"]), dtype=torch.float64, device="cuda")}
    if s["grad"]:
        out.update(dq=new("q"), dk=new("k"), dv=new("v"))
    a = b = 0
    for n, m in zip(s["lengths"], s["k_lengths"]):
        rows, keys = slice(a, a + n), slice(b, b + m)
        allowed = torch.ones((n, m), dtype=torch.bool, device="cuda")
        if s["causal"]:
            allowed = torch.tril(allowed, m - n)
        for h in range(s["q"].shape[1]):
            q, k, v = s["q"][rows, h].double(), s["k"][keys, h // group].double(), s["v"][keys, h // group].double()
            z = torch.where(allowed, q @ k.T / root, -math.inf)
            out["lse"][h, rows] = torch.logsumexp(z, 1)
            w = torch.softmax(z, 1)
            out["out"][rows, h] = w @ v
            if s["grad"]:  # the gradient of a softmax: w (g - sum w g)
                do = s["dout"][rows, h].double()
                g = do @ v.T
                g = w * (g - (w * g).sum(1, keepdim=True)) / root
                out["dq"][rows, h] = g @ k
                out["dk"][keys, h // group] += g.T @ q
                out["dv"][keys, h // group] += w.T @ do
        a, b = a + n, b + m
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "store":
        return {"k": _exact_block(s["k"]), "v": _exact_block(s["v"])}
    return {"rotate": _exact_rotate, "plan": _exact_plan, "cached": _exact_cached, "attend": _exact_attend}[case["op"]](s)
