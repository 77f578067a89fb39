"""The attention operators (include/tierstream_amd/tsa_attn.h) on an MI355X against plain implementations in 64 bits, at the sizes
and masks where they can go wrong: no token, one, tiles and pages that end anywhere, rows without keys, garbage behind the
last key, unaligned and unusual strides, every type and layout.

Tolerances in 2-norms of the whole result. Products of 16-bit values are exact in 32 bits and their sums are kept there: off by
about sqrt(n) 2^-24 of the terms, 2e-6 at the longest used here. A rounding to bf16 is off by 2^-8 / 2 / sqrt(3) = 1.2e-3 of the value in
the mean square, one to half precision by 1.5e-4. An output behind one rounded operand (probabilities, or the scores'
gradients) carries sqrt(2) of that, a gradient that also takes in the rounded output sqrt(3). The bounds are about twice those: 4e-3
(bf16), 5e-4 (f16), 1e-5 (f32, and a log sum of exponentials made of hardware's exponentials and logarithms)."""
import gc
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

KINDS = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BOUND = {torch.bfloat16: 4e-3, torch.float16: 5e-4, torch.float32: 1e-5}
PAGE = 64


@pytest.fixture(scope="module")
def attn(gpu):
    from tierstream_amd import attn
    yield attn
    gc.collect()              # graphs and tensors go now, not in the middle of another module's token,
    torch.cuda.synchronize()  # and the null stream is idle: streams of a device-gated context wait for what it still has


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def stream():
    return torch.cuda.current_stream().cuda_stream


def room(n):
    return torch.full((max(n, 16),), 0xFF, dtype=torch.uint8, device="cuda")


def near(got, want, what="", slack=0.0):
    assert got.shape == want.shape, what
    assert bool(torch.isfinite(got.double()).all()), f"{what}: not finite"
    norm, off = float(want.norm()), float((got.double() - want).norm())
    assert off <= BOUND[got.dtype] * norm + slack + 1e-30, f"{what}: off by {off / max(norm, 1e-30):.3g} of {norm:.3g}"


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def first_of(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return i32(at)


def rows(g, tokens, heads, dim, kind, layout="packed", sigma=1.0, fill=None):
    """[tokens][heads][dim], packed, inside wider rows of odd width ("odd"), heads first ("heads"), or as a slice of aligned rows."""
    t = KINDS[kind]
    if layout == "heads":
        x = torch.empty((heads, tokens, dim), dtype=t, device="cuda").transpose(0, 1)
    else:
        pad, shift = {"packed": (0, 0), "odd": (3, 1), "slice": (2, 1)}[layout]
        unit = 8 if layout == "slice" else 1
        flat = torch.full((tokens * (heads * dim + pad * unit) + shift * unit + 8,), 7.0, dtype=t, device="cuda")
        x = flat[shift * unit:].as_strided((tokens, heads, dim), (heads * dim + pad * unit, dim, 1))
    x.copy_(torch.randn((tokens, heads, dim), device="cuda", generator=g) * sigma if fill is None else torch.full((tokens, heads, dim), fill))
    return x


def replays(graph_of, check, n=4):
    """Captures graph_of(), and checks each replay, with eager work and waits between them."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph_of()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side, capture_error_mode="thread_local"):
        graph_of()
    for i in range(n):
        graph.replay()
        torch.cuda.synchronize()
        check(i)
        torch.randn(1000, device="cuda").sum().item()


# ---- rotate ------------------------------------------------------------------------------------------------------------------
def rotated64(x, positions, r, backward):
    """r: the Rotary."""
    n, y = r.s.pairs, x.double().clone()
    f = torch.tensor(list(r.s.turns)[:n], dtype=torch.float64, device="cuda") * 2 * math.pi
    angle = (positions.double()[:, None] * f)[:, None]
    a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if r.s.interleaved else (slice(0, n), slice(n, 2 * n))
    cos, sin = torch.cos(angle) * r.s.amplitude, torch.sin(angle) * r.s.amplitude * (-1 if backward else 1)
    p, q = y[..., a].clone(), y[..., b].clone()
    y[..., a], y[..., b] = p * cos - q * sin, p * sin + q * cos
    return y


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,kept,dim,rotated,layout", [
    (1, 1, 0, 2, 2, "packed"), (1, 32, 8, 128, 128, "packed"), (33, 5, 1, 64, 64, "slice"), (7, 4, 4, 80, 40, "packed"), (3, 2, 1, 256, 256, "packed"),
    (70, 3, 2, 96, 64, "heads"), (129, 2, 1, 72, 18, "odd"), (1000, 1, 1, 64, 16, "packed"), (5, 7, 0, 130, 130, "odd"), (2, 40, 8, 1024, 128, "slice")])
def test_rotate(attn, kind, interleaved, tokens, heads, kept, dim, rotated, layout):
    g = gen(tokens + heads)
    r = attn.Rotary(rotated, base=1e4, interleaved=interleaved, factor=4.0, trained=1024, amplitude=1.1)
    q, k = rows(g, tokens, heads, dim, kind, layout), rows(g, tokens, kept, dim, kind, layout) if kept else None
    positions = torch.randint(0, 1 << 20, (tokens,), device="cuda", generator=g, dtype=torch.int32)
    if tokens > 2:
        positions[1], positions[tokens - 1], positions[0] = 0, (1 << 31) - 1, -1
    live = positions >= 0
    for backward in (False, True):
        q_out, k_out = rows(g, tokens, heads, dim, kind, layout, fill=7.0), rows(g, tokens, kept, dim, kind, layout, fill=7.0) if kept else None
        attn.rotate(r, positions, q, k, q_out, k_out, backward=backward, stream=stream())
        for x, y in ((q, q_out), (k, k_out)):
            if x is not None:
                near(y[live], rotated64(x, positions, r, backward)[live])
                assert bool((y[~live] == 7).all()) and torch.equal(y[live][..., rotated:], x[live][..., rotated:])
                assert bool((x.untyped_storage() is not None))
    there, again = q.clone(), rows(g, tokens, heads, dim, kind, layout)
    again.copy_(q)
    attn.rotate(r, positions, again, stream=stream())
    q_out = torch.empty_like(there)
    q_out.copy_(there)
    attn.rotate(r, positions, there, None, q_out, stream=stream())
    assert torch.equal(again, q_out)  # in place is the same


def test_rotate_far_positions_keep_their_angle(attn):
    """At position 2^31 - 1 an angle in 32 bits would be off by 128 radians; in 64 by 2^-22, and products in 32 by 2^-23 of the pair."""
    r = attn.Rotary(128)
    x = torch.ones((2, 1, 128), device="cuda")
    positions = i32([(1 << 31) - 1, (1 << 31) - 2])
    y = torch.empty_like(x)
    attn.rotate(r, positions, x, None, y, stream=stream())
    assert float((y.double() - rotated64(x, positions, r, False)).abs().max()) < 2e-6


def test_rotate_gradient(attn):
    """<dy, R x> = <R^T dy, x>, and the difference quotient of a linear map is the map: sums of 2^14 terms in 32 bits."""
    g = gen(3)
    r = attn.Rotary(64, interleaved=True, amplitude=1.3)
    x, dy = (rows(g, 128, 2, 64, "f32") for _ in range(2))
    positions = torch.randint(0, 5000, (128,), device="cuda", generator=g, dtype=torch.int32)
    y, dx = torch.empty_like(x), torch.empty_like(x)
    attn.rotate(r, positions, x, None, y, stream=stream())
    attn.rotate(r, positions, dy, None, dx, backward=True, stream=stream())
    a, b = float((dy.double() * y.double()).sum()), float((dx.double() * x.double()).sum())
    assert abs(a - b) < 1e-5 * float(dy.norm()) * float(y.norm())


# ---- plan --------------------------------------------------------------------------------------------------------------------
def planned(lengths, fresh, table, free, n_free, n_rows, width):
    """The plan, request after request: everything it leaves, or the status."""
    pages = lambda n: (n + PAGE - 1) // PAGE  # noqa: E731
    table, free, count, status = [list(r) for r in table], list(free), n_free, 0
    need = gone = 0
    for n, f in zip(lengths, fresh):
        if n < 0:
            status |= 8
        elif f < 0:
            gone += pages(n)
            status |= 4 if pages(n) > width else 0
        elif pages(n + f) > width:
            status |= 4
        else:
            need += pages(n + f) - pages(n)
    if not 0 <= n_free <= len(free) or n_free + gone > len(free):
        status |= 8
    status |= 1 if need > n_free + gone else 0
    status |= 2 if sum(f for n, f in zip(lengths, fresh) if f > 0 and n >= 0) > n_rows else 0
    if status:
        return dict(ends=lengths, left=n_free, table=table, free=free, first=[0] * (len(lengths) + 1), positions=[-1] * n_rows, slots=[-1] * n_rows,
                    status=status)
    for i, f in enumerate(fresh):
        if f < 0:
            free[count:count + pages(lengths[i])] = table[i][:pages(lengths[i])]
            count += pages(lengths[i])
    ends, first, positions, slots = [], [0], [], []
    for i, (n, f) in enumerate(zip(lengths, fresh)):
        for p in range(pages(n), pages(n + f) if f > 0 else 0):
            count -= 1
            table[i][p] = free[count]
        for at in range(n, n + max(f, 0)):
            positions.append(at)
            slots.append(table[i][at // PAGE] * PAGE + at % PAGE)
        ends.append(0 if f < 0 else n + f)
        first.append(len(positions))
    rest = [-1] * (n_rows - len(positions))
    return dict(ends=ends, left=count, table=table, free=free, first=first, positions=positions + rest, slots=slots + rest, status=0)


def plan_case(seed, n, longest, n_rows, width, spare, kind):
    import random
    rng = random.Random(seed)
    lengths = [rng.choice([0, 1, 63, 64, 65, rng.randint(0, longest)]) for _ in range(n)]
    lengths = [min(v, longest) for v in lengths]
    if kind == "step":
        fresh = [1] * n
    else:
        fresh = [rng.choice([-1, 0, 1, 1, 2, 64, rng.randint(0, longest)]) for _ in range(n)]
        left = n_rows
        for i in range(n):
            fresh[i] = min(fresh[i], left) if fresh[i] > 0 else fresh[i]
            left -= max(fresh[i], 0)
    need = sum((v + 63) // 64 for v in lengths)
    numbers = list(range(need + spare))
    rng.shuffle(numbers)
    table = [[-7] * width for _ in range(n)]
    for i, v in enumerate(lengths):
        for p in range((v + 63) // 64):
            table[i][p] = numbers.pop()
    return lengths, fresh, table, numbers + [-9] * need, len(numbers)


def run_plan(attn, lengths, fresh, table, free, n_free, n_rows, width, in_place):
    n = len(lengths)
    new = lambda size: torch.full((size + 1,), 1234, dtype=torch.int32, device="cuda")  # noqa: E731
    wide = torch.full((max(n, 1), width + 3), 77, dtype=torch.int32, device="cuda")
    t = wide[:n, 1:1 + width]
    if n:
        t.copy_(i32(table))
    L, F, S, N = i32(lengths), i32(fresh), i32(free), i32([n_free])
    out = {k: new(v) for k, v in dict(ends=n, left=1, first=n + 1, positions=n_rows, slots=n_rows, status=1).items()}
    cut = {k: v[:-1] for k, v in out.items()}
    more = {} if in_place else dict(ends=cut["ends"], left=cut["left"])
    attn.plan(L, F, t, S, N, cut["first"], cut["positions"], cut["slots"], cut["status"], stream=stream(), **more)
    assert all(int(v[-1]) == 1234 for v in out.values())
    assert bool((wide[:, 0] == 77).all()) and bool((wide[:, 1 + width:] == 77).all())
    if in_place:
        cut["ends"], cut["left"] = L, N
    else:
        assert L.tolist() == lengths and N.tolist() == [n_free]
    got = {k: v.tolist() for k, v in cut.items()}
    got["left"], got["status"] = got["left"][0], got["status"][0]
    return dict(got, table=t.tolist(), free=S.tolist())


@pytest.mark.parametrize("seed,n,longest,n_rows,spare,kind", [
    (1, 1, 100, 1, 5, "step"), (2, 3, 1000, 40, 9, "step"), (3, 64, 500, 64, 70, "step"), (4, 7, 300, 400, 40, "mix"), (5, 100, 700, 3000, 200, "mix"),
    (6, 1025, 200, 9000, 1500, "mix"), (7, 4096, 130, 8192, 4096, "mix"), (8, 4095, 64, 4095, 4100, "step"), (9, 33, 3000, 8193, 600, "mix"), (10, 5, 90, 0, 5, "mix")])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan(attn, seed, n, longest, n_rows, spare, kind, in_place):
    width = 2 * longest // PAGE + 3
    case = plan_case(seed, n, longest, n_rows, width, spare, kind)
    want = planned(*case, n_rows, width)
    assert run_plan(attn, *case, n_rows, width, in_place) == want
    if kind == "step" or n_rows:
        assert want["status"] == 0 or n_rows == 0


@pytest.mark.parametrize("what,status", [("pages", 1), ("rows", 2), ("width", 4), ("length", 8), ("stack", 8), ("stack2", 8), ("ended", 8), ("two", 3)])
def test_plan_all_or_nothing(attn, what, status):
    lengths, fresh, n_rows, width, n_free = [64, 10, 130], [1, 100, -1], 120, 4, 6
    table = [[0, -1, -1, -1], [1, -1, -1, -1], [2, 3, 4, -1]]
    free = [5, 6, 7, 8, 9, 10] + [-1] * 4
    if what in ("pages", "two"):
        fresh, n_free, lengths = [1, 100, 0], 1, [64, 10, 130]
    if what in ("rows", "two"):
        n_rows = 50
    if what == "width":
        fresh[0] = 193
        n_rows = 400
    if what == "length":
        lengths[1] = -5
    if what == "stack":
        n_free = -1
    if what == "stack2":
        n_free = 11
    if what == "ended":
        n_free = 8  # three more than the stack has room for
    want = planned(lengths, fresh, table, free, n_free, n_rows, width)
    assert want["status"] == status
    assert run_plan(attn, lengths, fresh, table, free, n_free, n_rows, width, False) == want
    assert run_plan(attn, lengths, fresh, table, free, n_free, n_rows, width, True) == want


def test_plan_of_no_request(attn):
    want = planned([], [], [], [1, 2], 2, 5, 3)
    e = torch.empty(0, dtype=torch.int32, device="cuda")
    first, positions, slots, status, n_free = i32([9]), i32([9] * 5), i32([9] * 5), i32([9]), i32([2])
    attn.plan(e, e, torch.empty((0, 3), dtype=torch.int32, device="cuda"), i32([1, 2]), n_free, first, positions, slots, status, stream=stream())
    assert (first.tolist(), positions.tolist(), slots.tolist(), status.tolist(), n_free.tolist()) == ([0], want["positions"], want["slots"], [0], [2])


def test_slots(attn):
    """The rows of a plan once more; whole contexts; rows that have no page, or stand before the first token."""
    width, n_rows = 6, 300
    table = [[4, 2, 9, -1, -1, -1], [7, -1, -1, -1, -1, -1], [1 << 25, 3, -1, -1, -1, -1], [0, 5, 6, 8, 10, 11]]
    ends, counts = [130, 20, 70, 1000], [130, 20, 70, 5]  # the last ends behind its row's pages
    first, positions, slots = first_of(counts), i32([9] * n_rows), i32([9] * n_rows)
    attn.slots(i32(table), i32(ends), first, positions, slots, stream=stream())
    want_p, want_s = [], []
    for t, e, c in zip(table, ends, counts):
        for p in range(e - c, e):
            page = t[p // PAGE] if p // PAGE < width else -1
            want_p.append(p)
            want_s.append(page * PAGE + p % PAGE if 0 <= page < 1 << 25 else -1)
    rest = [-1] * (n_rows - len(want_p))
    assert positions.tolist() == want_p + rest and slots.tolist() == want_s + rest
    attn.slots(i32([[1, 2]]), i32([3]), i32([0, 5]), positions, slots, stream=stream())
    assert positions.tolist()[:6] == [-1, -1, 0, 1, 2, -1] and slots.tolist()[:6] == [-1, -1, 64, 65, 66, -1]


# ---- store and load ----------------------------------------------------------------------------------------------------------
def kept64(x):
    """What 4 bits leave of [..., n x 32] values."""
    b = x.double().unflatten(-1, (-1, 32))
    size = b.abs()
    at = (size == size.amax(-1, keepdim=True)).int().argmax(-1, keepdim=True)
    step = (torch.gather(b, -1, at) / -8).half().double()
    q = torch.where(step == 0, 0.0, torch.round(b / torch.where(step == 0, 1.0, step))).clamp(-8, 7)
    return (q * step).flatten(-2)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("tokens,kept,dim,layout", [(1, 1, 32, "packed"), (5, 8, 128, "packed"), (64, 3, 96, "slice"), (130, 2, 64, "odd"), (67, 4, 128, "heads"),
                                                    (700, 1, 128, "packed")])
def test_store_and_load(attn, kind, tokens, kept, dim, layout):
    g, n = gen(tokens), tokens // PAGE + 3
    pages = torch.randint(0, 256, (n, kept, 72 * dim), dtype=torch.uint8, device="cuda", generator=g)
    before, cache = pages.clone(), attn.Cache(pages, kept, dim)
    k, v = rows(g, tokens, kept, dim, kind, layout, 3.0), rows(g, tokens, kept, dim, kind, layout, 1e-3)
    if tokens > 4:
        k[1] = 0.0                      # no scale at all
        k[2, 0, :32] = 1.5              # every value of the largest size
        k[2, 0, 1], k[2, 0, 0] = -1.5, 0.5
        v[3] = v[3] * 1e-4              # scales below half precision's least
        k[4, 0, :32] = torch.arange(32, device="cuda") * 0.5 - 8.0   # ties: half steps
        v[0, 0, 5] = 60000.0
    slots = torch.randperm(n * PAGE, device="cuda", generator=g)[:tokens].to(torch.int32)
    if tokens > 60:
        slots[7], slots[8] = -1, n * PAGE  # skipped
    there = (slots >= 0) & (slots < n * PAGE)
    attn.store(cache, k, v, slots, stream=stream())
    k2, v2 = rows(g, tokens, kept, dim, kind, layout, fill=7.0), rows(g, tokens, kept, dim, kind, layout, fill=7.0)
    attn.load(cache, slots, k2, v2, stream=stream())
    for x, y in ((k, k2), (v, v2)):
        assert torch.equal(y[there], kept64(x).to(KINDS[kind])[there])
        assert bool((y[~there] == 7).all())
    # slots that were not given keep their bytes
    rest = torch.ones(n * PAGE, dtype=torch.bool, device="cuda")
    rest[slots[there].long()] = False
    nb = dim // 32
    for begin, width, shape, axis in ((0, 32 * dim, (n, kept, PAGE, 4 * nb * 4), 2), (32 * dim, 4 * dim, (n, kept, PAGE, nb * 2), 2),
                                      (36 * dim, 4 * dim, (n, kept, PAGE, nb * 2), 2), (40 * dim, 32 * dim, (n, kept, nb, PAGE, 16), 3)):
        a, b = (t[..., begin:begin + width].reshape(shape).movedim(axis, 1).reshape(n * PAGE, -1) for t in (before, pages))
        assert torch.equal(a[rest], b[rest])


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_blocks_that_hold_no_numbers_read_as_nan(attn, kind):
    pages = torch.zeros((1, 1, 72 * 64), dtype=torch.uint8, device="cuda")
    cache, k = attn.Cache(pages, 1, 64), torch.ones((4, 1, 64), dtype=KINDS[kind], device="cuda")
    k[0, 0, 3], k[1, 0, 40] = math.nan, math.inf
    if kind == "bf16":
        k[2, 0, 9] = 1e6  # its scale is beyond half precision
    attn.store(cache, k, k, i32([0, 1, 2, 3]), stream=stream())
    a, b = torch.empty_like(k), torch.empty_like(k)
    attn.load(cache, i32([0, 1, 2, 3]), a, b, stream=stream())
    bad = torch.zeros((4, 2), dtype=torch.bool, device="cuda")
    bad[0, 0] = bad[1, 1] = True
    bad[2, 0] = kind == "bf16"
    for t in (a, b):
        assert torch.equal(t.view(4, 2, 32).isnan().all(2), bad) and torch.equal(t.view(4, 2, 32).isnan().any(2), bad)


# ---- attention over the cache ------------------------------------------------------------------------------------------------
def numbers64(pages, dim):
    """Keys and values [2][n][heads][64][dim] of pages."""
    n, kept, nb = pages.shape[0], pages.shape[1], dim // 32
    keys = pages[..., :32 * dim].view(n, kept, PAGE, 4, nb, 4).transpose(3, 4).reshape(n, kept, PAGE, nb, 16)
    values = pages[..., 40 * dim:].view(n, kept, nb, PAGE, 16).transpose(2, 3)
    scales = pages[..., 32 * dim:40 * dim].contiguous().view(torch.float16).double().view(n, kept, 2, PAGE, nb, 1)
    out = [torch.cat([x & 15, x >> 4], -1).double() - 8 for x in (keys, values)]
    return torch.stack([(x * scales[:, :, i]).flatten(-2) for i, x in enumerate(out)])


def random_pages(g, n, kept, dim, sigma=(0.25, 0.1)):
    pages = torch.randint(0, 256, (n, kept, 72 * dim), dtype=torch.uint8, device="cuda", generator=g)
    for i in range(2):
        s = (torch.randn((n, kept, 2 * dim), device="cuda", generator=g) * sigma[i]).half()
        pages[..., (32 + 4 * i) * dim:(36 + 4 * i) * dim] = s.view(torch.uint8)
    return pages


def cached64(q, pages, dim, table, ends, counts, scale, n_pages):
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    group, at = q.shape[1] // pages.shape[1], 0
    for i, c in enumerate(counts):
        end = min(ends[i], table.shape[1] * PAGE)
        used = table[i, :(max(end, 0) + PAGE - 1) // PAGE].long()
        there = (used >= 0) & (used < n_pages)
        k, v = numbers64(pages[used.clamp(0, n_pages - 1)], dim).transpose(1, 2).reshape(2, pages.shape[1], -1, dim)  # [heads][tokens][dim]
        there = there.repeat_interleave(PAGE)
        for t in range(c):
            seen = there & (torch.arange(len(there), device="cuda") < end - c + t + 1)
            for h in range(q.shape[1]):
                kk, vv = k[h // group][seen], v[h // group][seen]
                if len(kk):
                    out[at + t, h] = torch.softmax(kk @ q[at + t, h].double() * scale, 0) @ vv
        at += c
    return out


CACHED = [  # ends, fresh, kept, group, dim
    ([1], [1], 1, 1, 32), ([64], [1], 2, 4, 128), ([65], [1], 8, 4, 128), ([63, 1, 128, 700], [1] * 4, 4, 8, 128), ([2100], [1], 1, 16, 64),
    ([5, 300], [5, 2], 2, 5, 96), ([200, 0, 77], [3, 0, 8], 2, 1, 64), ([1000, 130], [1, 0], 3, 3, 128), ([4099], [4], 2, 4, 128), ([90], [40], 1, 6, 128),
    ([3], [5], 2, 2, 64), ([129, 64, 65, 63, 1, 2, 192, 500, 3], [1] * 9, 2, 2, 32), ([300], [17], 1, 33, 64),
    ([9000, 17000], [1, 2], 8, 4, 128), ([20001], [1], 8, 2, 64), ([700] * 12, [2] * 12, 16, 1, 96)]  # (thousands of pages)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("ends,fresh,kept,group,dim", CACHED)
@pytest.mark.parametrize("layout", ["packed", "odd"])
def test_attend_cached(attn, kind, ends, fresh, kept, group, dim, layout):
    g, tokens = gen(sum(ends)), sum(fresh)
    need = [(e + PAGE - 1) // PAGE for e in ends]
    n, width = sum(need) + 2, max(need) + 1
    pages = random_pages(g, n, kept, dim)
    order, at = torch.randperm(n, device="cuda", generator=g).tolist(), 0
    wide = torch.full((len(ends), width + 2), 1 << 30, dtype=torch.int32, device="cuda")  # behind a request's pages: garbage
    table = wide[:, :width]
    for i, p in enumerate(need):
        table[i, :p] = i32(order[at:at + p])
        at += p
        if ends[i] % PAGE:  # behind the last key: NaN scales
            last = pages[order[at - 1]]
            for part in range(2):
                last[:, (32 + 4 * part) * dim:(36 + 4 * part) * dim].view(kept, PAGE, -1)[:, ends[i] % PAGE:] = 0xFF
    q = rows(g, tokens + 2, kept * group, dim, kind, layout)
    out = rows(g, tokens + 2, kept * group, dim, kind, layout, fill=7.0)
    cache, e, f = attn.Cache(pages, kept, dim), i32(ends), first_of(fresh)
    ws = room(attn.attend_cached_workspace(cache, q, table))
    attn.attend_cached(cache, q, out, table, e, f, scale=0.2, workspace=ws, stream=stream())
    want = cached64(q[:tokens], pages, dim, table, ends, fresh, 0.2, n)
    near(out[:tokens], want)
    assert bool((out[tokens:] == 7).all())
    again = rows(g, tokens + 2, kept * group, dim, kind, layout, fill=7.0)
    attn.attend_cached(cache, q, again, table, e, f, scale=0.2, workspace=ws, stream=stream())
    assert torch.equal(out, again)


@pytest.mark.parametrize("ends", [[200, 500, 100], [-5, 1 << 30, 0]])
def test_attend_cached_reads_no_page_out_of_range(attn, ends):
    """Absent pages count as absent, lengths end at the table; a request none of whose pages are there gives 0."""
    g = gen(9)
    pages = random_pages(g, 12, 2, 64)
    table = i32([[0, -1, 2, 12, 3, 4, 5, 1 << 30], [-1] * 8, [6, 7, 8, 9, 10, 11, 1, 2]])
    q, out = rows(g, 3, 4, 64, "bf16"), rows(g, 3, 4, 64, "bf16", fill=7.0)
    cache = attn.Cache(pages, 2, 64)
    attn.attend_cached(cache, q, out, table, i32(ends), i32([0, 1, 2, 3]), workspace=room(attn.attend_cached_workspace(cache, q, table)), stream=stream())
    near(out, cached64(q, pages, 64, table, ends, [1, 1, 1], 0.125, 12))
    assert bool((out[1] == 0).all())


def test_attend_cached_large_scores(attn):
    """Scores far apart: the running maximum, in both directions."""
    g = gen(4)
    for sigma in (30.0, 1e-6):
        pages = random_pages(g, 20, 1, 128, (sigma, 0.1))
        table = torch.arange(20, device="cuda", dtype=torch.int32)[None]
        q, out = rows(g, 1, 8, 128, "f16"), torch.empty((1, 8, 128), dtype=torch.float16, device="cuda")
        cache = attn.Cache(pages, 1, 128)
        attn.attend_cached(cache, q, out, table, i32([1277]), i32([0, 1]), workspace=room(attn.attend_cached_workspace(cache, q, table)), stream=stream())
        # a score of size s is off by 2^-24 s sqrt(128) at most, and so is its probability, relatively
        near(out, cached64(q, pages, 128, table, [1277], [1], 128 ** -0.5, 20), slack=(1e-3 if sigma > 1 else 0) * float(out.double().norm()))


@pytest.mark.parametrize("value", [1e-7, 4e-4, 3000.0])
def test_attend_cached_scales_of_values(attn, value):
    """Half precision's own range does not limit what lies between (the smallest scales are its subnormals, exact in the cache)."""
    g = gen(6)
    pages = random_pages(g, 10, 2, 64, (0.2, value))
    table = torch.arange(10, device="cuda", dtype=torch.int32)[None]
    q, out = rows(g, 1, 4, 64, "f16"), torch.empty((1, 4, 64), dtype=torch.float16, device="cuda")
    cache = attn.Cache(pages, 2, 64)
    attn.attend_cached(cache, q, out, table, i32([640]), i32([0, 1]), workspace=room(attn.attend_cached_workspace(cache, q, table)), stream=stream())
    want = cached64(q, pages, 64, table, [640], [1], 0.125, 10)
    # an output below half precision's normal numbers is off by half of its least step
    near(out, want, slack=2.0 ** -25 * math.sqrt(out.numel()))


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_attend_cached_scales_of_values_far_apart(attn, kind):
    """Largest scales that grow from page to page, small ones beside them, and blocks of very different ones; scores that pick few tokens."""
    g = gen(16)
    for sigma in (0.2, 6.0):
        pages = random_pages(g, 40, 2, 64, (sigma, 0.1))
        scales = pages[..., 36 * 64:40 * 64].view(torch.float16).view(40, 2, PAGE, 2)
        by = torch.exp2(-torch.randint(0, 13, scales.shape, device="cuda", generator=g).float())
        by *= torch.exp2(torch.arange(40, device="cuda")[:, None, None, None] / 5)
        by[..., 1] *= 2.0 ** -8
        scales *= by.half()
        table = torch.arange(40, device="cuda", dtype=torch.int32)[None]
        q, out = rows(g, 2, 6, 64, kind), torch.empty((2, 6, 64), dtype=KINDS[kind], device="cuda")
        cache = attn.Cache(pages, 2, 64)
        attn.attend_cached(cache, q, out, table, i32([2500]), i32([0, 2]), workspace=room(attn.attend_cached_workspace(cache, q, table)), stream=stream())
        want = cached64(q, pages, 64, table, [2500], [2], 0.125, 40)
        for b in range(2):  # (each by itself: the second is 2^8 smaller)
            near(out[..., 32 * b:32 * b + 32], want[..., 32 * b:32 * b + 32])


@pytest.mark.parametrize("scale", [-0.3, 0.0, -0.0, 1e-38])
def test_attend_cached_scale_of_any_sign(attn, scale):
    g = gen(17)
    pages = random_pages(g, 8, 2, 96)
    table = i32([[3, 1, 0, 7, 2], [4, 5, 6, -1, -1]])
    q, out = rows(g, 5, 4, 96, "f16"), torch.empty((5, 4, 96), dtype=torch.float16, device="cuda")
    cache, ends, fresh = attn.Cache(pages, 2, 96), [290, 129], [2, 3]
    attn.attend_cached(cache, q, out, table, i32(ends), first_of(fresh), scale=scale, workspace=room(attn.attend_cached_workspace(cache, q, table)), stream=stream())
    near(out, cached64(q, pages, 96, table, ends, fresh, scale, 8))


@pytest.mark.parametrize("requests", [257, 700, 1025, 4096])
def test_attend_cached_of_many_requests(attn, requests):
    """Most of a page or two, some without new tokens, one long and in pieces, wherever it stands."""
    g = gen(requests)
    pages = random_pages(g, 70, 1, 32)
    ends = torch.randint(1, 100, (requests,), device="cuda", generator=g).tolist()
    fresh = [int(i % 7 != 3) for i in range(requests)]
    for long in (0, requests // 2 + 1, requests - 1):
        ends[long], fresh[long] = 60 * PAGE + 5, 3
    table = torch.randint(0, 70, (requests, 61), device="cuda", generator=g, dtype=torch.int32)
    q = rows(g, sum(fresh), 8, 32, "f16")
    out, cache = torch.empty_like(q), attn.Cache(pages, 1, 32)
    attn.attend_cached(cache, q, out, table, i32(ends), first_of(fresh), workspace=room(attn.attend_cached_workspace(cache, q, table)), stream=stream())
    near(out, cached64(q, pages, 32, table, ends, fresh, 32 ** -0.5, 70))


# ---- attention over packed sequences -----------------------------------------------------------------------------------------
def attend64(q, k, v, counts, k_counts, causal, scale, dout=None):
    group = q.shape[1] // k.shape[1]
    out, lse = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.full((q.shape[1], q.shape[0]), -math.inf, dtype=torch.float64, device="cuda")
    dq, dk, dv = (torch.zeros(t.shape, dtype=torch.float64, device="cuda") for t in (q, k, v))
    a = b = 0
    for n, m in zip(counts, k_counts):
        ok = torch.ones((n, m), dtype=torch.bool, device="cuda")
        if causal:
            ok = torch.tril(ok, m - n)
        for h in range(q.shape[1]):
            kh = h // group
            x, y, z = q[a:a + n, h].double(), k[b:b + m, kh].double(), v[b:b + m, kh].double()
            s = (x @ y.T * scale).masked_fill(~ok, -math.inf)
            p = torch.softmax(s, 1).nan_to_num(0.0) if m else torch.zeros((n, 0), dtype=torch.float64, device="cuda")
            out[a:a + n, h] = p @ z
            lse[h, a:a + n] = torch.logsumexp(s, 1) if m else -math.inf
            if dout is not None:
                d = dout[a:a + n, h].double()
                gr = d @ z.T
                ds = p * (gr - (p * gr).sum(1, keepdim=True)) * scale
                dq[a:a + n, h], dk[b:b + m, kh], dv[b:b + m, kh] = ds @ y, dk[b:b + m, kh] + ds.T @ x, dv[b:b + m, kh] + p.T @ d
        a, b = a + n, b + m
    return out, lse, dq, dk, dv


ATTEND = [  # queries, keys (None: as many), kept, group, dim
    ([1], None, 1, 1, 64), ([64], None, 2, 2, 128), ([65], None, 1, 4, 128), ([1, 2, 3, 127, 128, 129], None, 2, 1, 64), ([300], None, 1, 2, 72),
    ([33, 0, 200], None, 2, 3, 8), ([10, 70], [300, 5], 2, 2, 128), ([40], [40 + 512], 1, 4, 64), ([5, 64], [0, 64], 1, 1, 32), ([257, 31], None, 4, 1, 104),
    ([513], None, 1, 1, 128), ([1, 1, 1, 1], [1, 64, 65, 1000], 2, 4, 128), ([5] * 70, None, 1, 2, 64),
    ([300, 77], None, 2, 4, 128), ([1, 600], [70, 650], 4, 2, 64), ([190, 3, 130], [260, 64, 100], 1, 8, 72)]  # (more rows than take both parts)


def attend_case(kind, counts, k_counts, kept, group, dim, layout, pad=3):
    g = gen(sum(counts) * 7 + dim)
    k_counts = counts if k_counts is None else k_counts
    t, m = sum(counts) + pad, sum(k_counts) + pad
    q, k, v = rows(g, t, kept * group, dim, kind, layout), rows(g, m, kept, dim, kind, layout), rows(g, m, kept, dim, kind, layout)
    dout = rows(g, t, kept * group, dim, kind, layout, 0.1)
    for x, n in ((q, t), (k, m), (v, m), (dout, t)):
        x[n - pad:] = math.nan  # behind the last sequence
    return q, k, v, dout, k_counts, first_of(counts), first_of(k_counts)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("counts,k_counts,kept,group,dim", ATTEND)
@pytest.mark.parametrize("layout", ["packed", "odd"])
def test_attend_and_its_gradients(attn, kind, causal, counts, k_counts, kept, group, dim, layout):
    q, k, v, dout, k_counts, first, k_first = attend_case(kind, counts, k_counts, kept, group, dim, layout)
    t, m, scale = sum(counts), sum(k_counts), 0.9 * dim ** -0.5
    fresh = lambda x: rows(None, *x.shape, kind, layout, fill=7.0)  # noqa: E731
    out, lse = fresh(q), torch.full((kept * group, len(q)), 7.0, device="cuda")
    where = dict(first=first, k_first=k_first, causal=causal, scale=scale, stream=stream())
    attn.attend(q, k, v, out, lse=lse, **where)
    want = attend64(q[:t], k[:m], v[:m], counts, k_counts, causal, scale, dout[:t])
    near(out[:t], want[0], "out")
    live = ~torch.isinf(want[1])
    near(lse[:, :t][live], want[1][live], "lse")
    assert bool((lse[:, :t][~live] == -math.inf).all()) and bool((out[:t].transpose(0, 1)[~live] == 0).all())
    assert bool((out[t:] == 7).all()) and bool((lse[:, t:] == 7).all())
    dq, dk, dv = fresh(q), fresh(k), fresh(v)
    ws = room(attn.attend_backward_workspace(q, k))
    attn.attend_backward(q, k, v, out, dout, lse, dq, dk, dv, workspace=ws, **where)
    # a sequence of one key has score gradients of 0, made of a difference of two sums of dim products that are rounded in 32 bits, and of
    # what rounding the output leaves: 2^-9 of a term each
    small = BOUND[q.dtype] / 4 * float(dout[:t].double().norm()) * float(v[:m].double().norm(dim=-1).max() if m else 0) * scale
    for name, got, exact, n, other in (("dq", dq, want[2], t, k[:m]), ("dk", dk, want[3], m, q[:t]), ("dv", dv, want[4], m, None)):
        near(got[:n], exact, name, slack=0.0 if other is None or not len(other) else small * float(other.double().abs().max()) * 0.05)
        assert bool((got[n:] == 7).all()), name
    dq2, dk2, dv2 = fresh(q), fresh(k), fresh(v)
    attn.attend_backward(q, k, v, out, dout, lse, dq2, workspace=ws, **where)
    attn.attend_backward(q, k, v, out, dout, lse, None, dk2, dv2, workspace=ws, **where)
    assert torch.equal(dq, dq2) and torch.equal(dk, dk2) and torch.equal(dv, dv2)  # asked for apart, and the same bits again


def test_attend_one_sequence_without_first(attn):
    q, k, v, _, _, first, k_first = attend_case("bf16", [100], [150], 2, 2, 64, "packed", pad=0)
    a, b = torch.empty_like(q), torch.empty_like(q)
    attn.attend(q, k, v, a, stream=stream())
    attn.attend(q, k, v, b, first=first, k_first=k_first, stream=stream())
    assert torch.equal(a, b)


@pytest.mark.parametrize("layouts", [("slice", "heads"), ("heads", "packed")])
def test_attend_takes_slices_and_shared_heads(attn, layouts):
    """Queries, keys and values as slices of one product; heads first; one key head for all by a stride of 0."""
    g, t, dim = gen(1), 140, 64
    one = rows(g, t, 8, dim, "bf16", layouts[0])
    q, k, v = one[:, :4], one[:, 4:6], one[:, 6:]
    out = rows(g, t, 4, dim, "bf16", layouts[1], fill=0.0)
    attn.attend(q, k, v, out, stream=stream())
    near(out, attend64(q, k, v, [t], [t], True, dim ** -0.5)[0])
    shared = k[:, :1].expand(t, 4, dim)
    attn.attend(q, shared, shared, out, stream=stream())
    near(out, attend64(q, shared, shared, [t], [t], True, dim ** -0.5)[0])


def test_attend_takes_sequences_as_they_are(attn):
    """first that is not ascending, or goes beyond the rows, reads and writes nothing out of range: what is inside is right."""
    q, k, v, dout, _, _, _ = attend_case("bf16", [128], None, 1, 1, 64, "packed", pad=0)
    for first in ([0, 50, 40, 1000], [-5, 50, 50, 1 << 30], [60, 20, 128, 128]):
        f, out, lse = i32(first), torch.full_like(q, 7.0), torch.zeros((1, 128), device="cuda")
        attn.attend(q, k, v, out, lse=lse, first=f, stream=stream())
        grads = [torch.full_like(x, 7.0) for x in (q, k, v)]
        attn.attend_backward(q, k, v, out, dout, lse, *grads, first=f, workspace=room(attn.attend_backward_workspace(q, k)), stream=stream())
        assert bool(torch.isfinite(out.float()).all()) and all(bool(torch.isfinite(x.float()).all()) for x in grads)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_infinities_stay_in_the_rows_that_attend_to_them(attn, kind):
    q, k, v, dout, _, first, _ = attend_case(kind, [200, 130], None, 1, 2, 64, "packed", pad=0)
    k[150], v[160, 0, 3], q[20, 1] = math.nan, math.inf, math.inf
    out, lse = torch.empty_like(q), torch.empty((2, 330), device="cuda")
    attn.attend(q, k, v, out, lse=lse, first=first, stream=stream())
    ok = torch.ones((330, 2), dtype=torch.bool, device="cuda")
    ok[150:200] = False
    ok[20, 1] = False
    k2, v2, q2 = k.clone(), v.clone(), q.clone()
    k2[150], v2[160], q2[20, 1] = 0, 0, 0
    want = attend64(q2, k2, v2, [200, 130], [200, 130], True, 0.125)[0]
    near(out[ok], want[ok])
    dq, dk, dv = (torch.empty_like(x) for x in (q, k, v))
    attn.attend_backward(q, k, v, out, dout, lse, dq, dk, dv, first=first, workspace=room(attn.attend_backward_workspace(q, k)), stream=stream())
    assert bool(torch.isfinite(dq[ok].float()).all()) and bool(torch.isfinite(dk[200:].float()).all()) and bool(torch.isfinite(dv[200:].float()).all())


def rounded_output(q, k, want_out, dout, counts, scale, eps):
    """What rounding the output to 16 bits adds to the gradients. The backward pass takes sum_j p_j dp_j = dout . out from the rounded output:
    off by d_t = sum_i dout_ti out_ti e_ti, |e| <= eps / 2, at most eps / 2 |dout_t * out_t| in the 2-norm over independent e. Each
    ds_tj = scale p_tj (dp_tj - sum) is off by scale p_tj d_t, so dq_t by scale d_t sum_j p_tj k_j and dk_j by scale sum_t p_tj d_t q_t. Where one
    probability is nearly 1 the difference itself is nearly 0, and these terms are what is left. One head, causal."""
    d, dq2, dk2, a = eps / 2 * (dout.double() * want_out)[:, 0].norm(dim=1), 0.0, 0.0, 0
    for n in counts:
        x, y = q[a:a + n, 0].double(), k[a:a + n, 0].double()
        p = torch.softmax((x @ y.T * scale).masked_fill(~torch.tril(torch.ones((n, n), dtype=torch.bool, device="cuda")), -math.inf), 1)
        dq2 += float(((d[a:a + n] * scale) ** 2 * (p @ y).square().sum(1)).sum())
        dk2 += float(((p * (d[a:a + n] * scale * x.norm(dim=1))[:, None]) ** 2).sum())
        a += n
    return math.sqrt(dq2), math.sqrt(dk2)


def test_attend_large_scores(attn):
    """Scores of some hundred either way, and a key far above all others in the last tile."""
    q, k, v, dout, _, _, _ = attend_case("f16", [400], None, 1, 1, 128, "packed", pad=0)
    k[390] = q[395, 0] * 2
    for s in (1.0, 8.0):
        out, lse = torch.empty_like(q), torch.empty((1, 400), device="cuda")
        attn.attend(q, k, v, out, lse=lse, scale=s, stream=stream())
        want = attend64(q, k, v, [400], [400], True, s, dout)
        # a score of size x is off by 2^-24 x a few, and so is its probability, relatively
        near(out, want[0], slack=1e-4 * s * float(want[0].norm()))
        near(lse, want[1])
        dq, dk, dv = (torch.empty_like(x) for x in (q, k, v))
        attn.attend_backward(q, k, v, out, dout, lse, dq, dk, dv, scale=s, workspace=room(attn.attend_backward_workspace(q, k)), stream=stream())
        more = rounded_output(q, k, want[0], dout, [400], s, torch.finfo(torch.float16).eps)
        for got, exact, add in zip((dq, dk, dv), want[2:], (*more, 0.0)):
            near(got, exact, slack=2e-4 * s * float(exact.norm()) + add)


@pytest.mark.parametrize("sigma", [1e-6, 1e-3, 300.0])
def test_half_precision_gradients_of_any_size(attn, sigma):
    """Gradients of the scores may lie far below half precision's normal numbers, or above its largest."""
    q, k, v, dout, _, first, _ = attend_case("f16", [150, 90], None, 2, 2, 64, "packed", pad=0)
    dout = (dout.double() * 10 * sigma).half()
    v.mul_(4)
    out, lse = torch.empty_like(q), torch.empty((4, 240), device="cuda")
    attn.attend(q, k, v, out, lse=lse, first=first, stream=stream())
    dq, dk, dv = (torch.empty_like(x) for x in (q, k, v))
    attn.attend_backward(q, k, v, out, dout, lse, dq, dk, dv, first=first, workspace=room(attn.attend_backward_workspace(q, k)), stream=stream())
    want = attend64(q, k, v, [150, 90], [150, 90], True, 0.125, dout)
    for got, exact in zip((dq, dk, dv), want[2:]):
        near(got, exact, slack=2.0 ** -25 * math.sqrt(got.numel()))  # the output's own least step


def test_gradients_against_differences(attn):
    """(f(x + h u) - f(x - h u)) / 2 h against <gradient, u>, f = sum out x dout. The differences are taken of the 64-bit formula, at
    h = 1e-4 where they are right to 1e-6; the gradients are the operator's."""
    q, k, v, dout, _, first, _ = attend_case("bf16", [70, 50], None, 2, 2, 64, "packed", pad=0)
    out, lse = torch.empty_like(q), torch.empty((4, 120), device="cuda")
    attn.attend(q, k, v, out, lse=lse, first=first, stream=stream())
    grads = [torch.empty_like(x) for x in (q, k, v)]
    attn.attend_backward(q, k, v, out, dout, lse, *grads, first=first, workspace=room(attn.attend_backward_workspace(q, k)), stream=stream())
    g, at = gen(5), [x.double() for x in (q, k, v)]
    f = lambda xs: float((attend64(*xs, [70, 50], [70, 50], True, 0.125)[0] * dout.double()).sum())  # noqa: E731
    for i in range(3):
        u = torch.randn(at[i].shape, device="cuda", generator=g, dtype=torch.float64)
        up, down = list(at), list(at)
        up[i], down[i] = at[i] + 1e-4 * u, at[i] - 1e-4 * u
        slope, want = (f(up) - f(down)) / 2e-4, float((grads[i].double() * u).sum())
        assert abs(slope - want) <= BOUND[torch.bfloat16] * float(grads[i].double().norm()) * 4, (i, slope, want)


def test_backward_captured_while_an_eager_graph_lives(attn):
    """Forward and backward passes captured and replayed, on another stream, beside an eager autograd graph of the same leaves."""
    q, k, v, dout, _, first, _ = attend_case("bf16", [90, 200], None, 2, 2, 64, "packed", pad=0)
    leaf = q.float().requires_grad_()
    alive = (leaf * 2).sum()
    out, lse = torch.empty_like(q), torch.empty((4, 290), device="cuda")
    grads, ws = [torch.empty_like(x) for x in (q, k, v)], room(attn.attend_backward_workspace(q, k))
    attn.attend(q, k, v, out, lse=lse, first=first, stream=stream())
    attn.attend_backward(q, k, v, out, dout, lse, *grads, first=first, workspace=ws, stream=stream())
    want = [x.clone() for x in (out, lse, *grads)]

    def both():
        attn.attend(q, k, v, out, lse=lse, first=first, stream=stream())
        attn.attend_backward(q, k, v, out, dout, lse, *grads, first=first, workspace=ws, stream=stream())

    def check(i):
        assert all(torch.equal(a, b) for a, b in zip((out, lse, *grads), want)), i
        for x in (out, lse, *grads):
            x.fill_(0)

    replays(both, check)
    alive.backward()
    assert bool((leaf.grad == 2).all())


# ---- together ----------------------------------------------------------------------------------------------------------------
def test_a_decode_loop(attn):
    """Prompts, then steps of one captured graph (plan, rotate, store, attend) over requests that come and go: each step against
    the rotated keys and values that 4 bits leave, kept apart by the test."""
    g, kept, group, dim, width, n_pages, n, capacity = gen(8), 2, 4, 64, 5, 14, 4, 130
    heads, r = kept * group, attn.Rotary(64, base=1e4)
    pages = torch.full((n_pages, kept, 72 * dim), 0xFF, dtype=torch.uint8, device="cuda")
    cache = attn.Cache(pages, kept, dim)
    new = lambda *shape: torch.zeros(shape, dtype=torch.int32, device="cuda")  # noqa: E731
    lengths, fresh, table, free, n_free = new(n), new(n), new(n, width), torch.arange(n_pages, device="cuda", dtype=torch.int32), i32([n_pages])
    first, positions, slots, status = new(n + 1), new(capacity), new(capacity), new(1)
    q, k, v = (torch.zeros((capacity, h, dim), dtype=torch.bfloat16, device="cuda") for h in (heads, kept, kept))
    out = torch.zeros_like(q)
    ws = room(attn.attend_cached_workspace(cache, q, table))

    def step():
        attn.plan(lengths, fresh, table, free, n_free, first, positions, slots, status, stream=stream())
        attn.rotate(r, positions, q, k, stream=stream())
        attn.store(cache, k, v, slots, stream=stream())
        attn.attend_cached(cache, q, out, table, lengths, first, workspace=ws, stream=stream())

    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side, capture_error_mode="thread_local"):
        step()
    held = [[] for _ in range(n)]  # each request's (keys, values) as 4 bits leave them
    for asked in ([70, 3, 0, 1], [1, 1, 40, 1], [1, 64, 1, 1], [-1, 1, 1, 1], [100, -1, 1, 0], [1, 30, 1, 1], [1, 1, 1, 62], [1, 1, 1, 1], [1, 1, -1, 2]):
        used = sum(max(a, 0) for a in asked)
        fresh.copy_(i32(asked))
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, device="cuda", generator=g))
        raw_q, raw_k, raw_v = q.clone(), k.clone(), v.clone()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert int(status) == 0 and int(first[-1]) == used and bool((positions[used:] == -1).all())
        assert torch.equal(q[used:], raw_q[used:])
        at = 0
        for i, a in enumerate(asked):
            if a < 0:
                held[i] = []
            for t in range(max(a, 0)):
                p = i32([len(held[i])])
                assert int(positions[at]) == len(held[i])
                key = k[at:at + 1]
                near(key, rotated64(raw_k[at:at + 1], p, r, False))
                held[i].append((kept64(key)[0], kept64(raw_v[at:at + 1])[0]))
                kk, vv = (torch.stack([pair[j] for pair in held[i]]) for j in range(2))  # [tokens][kept][dim]
                for h in range(heads):
                    w = torch.softmax(kk[:, h // group] @ q[at, h].double() * dim ** -0.5, 0)
                    near(out[at, h], w @ vv[:, h // group], slack=4e-3 * float(vv.abs().max()))
                at += 1
        assert lengths.tolist() == [len(x) for x in held]
        live = [p for i in range(n) for p in table[i, :(len(held[i]) + 63) // 64].tolist()]
        assert sorted(live + free[:int(n_free)].tolist()) == list(range(n_pages))  # every page once


def test_two_streams_with_workspaces_of_their_own(attn):
    """Two calls at once, and two captured graphs that are replayed one after the other over one workspace."""
    g = gen(2)
    pages = random_pages(g, 40, 2, 128)
    cache, table = attn.Cache(pages, 2, 128), torch.arange(40, device="cuda", dtype=torch.int32).view(2, 20)
    ends, first = i32([1280, 1201]), i32([0, 1, 2])
    qs = [rows(g, 2, 8, 128, "bf16") for _ in range(2)]
    need = attn.attend_cached_workspace(cache, qs[0], table)
    want = []
    for q in qs:
        want.append(torch.empty_like(q))
        attn.attend_cached(cache, q, want[-1], table, ends, first, workspace=room(need), stream=stream())
    torch.cuda.synchronize()
    streams, got, rooms = [torch.cuda.Stream() for _ in qs], [torch.zeros_like(q) for q in qs], [room(need) for _ in qs]
    for s, q, o, w in zip(streams, qs, got, rooms):
        s.wait_stream(torch.cuda.current_stream())
        for _ in range(20):
            attn.attend_cached(cache, q, o, table, ends, first, workspace=w, stream=s.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, one = [], room(need)
    for q, o in zip(qs, got):
        o.zero_()
        graphs.append(torch.cuda.CUDAGraph())
        torch.cuda.synchronize()
        with torch.cuda.graph(graphs[-1], stream=streams[0], capture_error_mode="thread_local"):
            attn.attend_cached(cache, q, o, table, ends, first, workspace=one, stream=stream())
    for _ in range(3):
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        for o in got:
            o.zero_()


def test_nothing_of_no_token(attn):
    r, e = attn.Rotary(64), torch.empty((0, 2, 64), dtype=torch.bfloat16, device="cuda")
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    attn.rotate(r, none, e, e, stream=stream())
    cache = attn.Cache(torch.empty((0, 2, 72 * 64), dtype=torch.uint8, device="cuda"), 2, 64)
    attn.store(cache, e, e, none, stream=stream())
    attn.load(cache, none, e, e, stream=stream())
    attn.attend(e, e, e, e, stream=stream())
    q, out = torch.ones((3, 2, 64), dtype=torch.bfloat16, device="cuda"), torch.ones((3, 2, 64), dtype=torch.bfloat16, device="cuda")
    lse = torch.zeros((2, 3), device="cuda")
    attn.attend(q, e, e, out, lse=lse, stream=stream())  # no key: zeros
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    dq = torch.ones_like(q)
    attn.attend_backward(q, e, e, out, q, lse, dq, e, e, workspace=room(attn.attend_backward_workspace(q, e)), stream=stream())
    assert bool((dq == 0).all())
    dk, dv = torch.ones_like(q), torch.ones_like(q)
    attn.attend_backward(e, q, q, e, e, torch.empty((2, 0), device="cuda"), e, dk, dv, workspace=room(attn.attend_backward_workspace(e, q)), stream=stream())
    assert bool((dk == 0).all()) and bool((dv == 0).all())  # keys without a query


# ---- what the documents allow beyond that ------------------------------------------------------------------------------------
@pytest.mark.parametrize("first", [[0, 2, 1, 9], [-4, 1, 3, 1 << 30], [3, 0, 0, 3], [5, 5, 5, 5]])
def test_attend_cached_takes_requests_as_they_are(attn, first):
    """first that is not ascending, or goes beyond the rows: nothing out of range is read or written."""
    g = gen(31)
    pages = random_pages(g, 12, 1, 64)
    table = torch.arange(12, device="cuda", dtype=torch.int32).view(3, 4)
    whole = torch.full((9, 4, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    q, out = rows(g, 3, 4, 64, "bf16"), whole[3:6]
    cache = attn.Cache(pages, 1, 64)
    size = attn.attend_cached_workspace(cache, q, table)
    ws = torch.full((size + 1024,), 99, dtype=torch.uint8, device="cuda")
    attn.attend_cached(cache, q, out, table, i32([250, 200, 256]), i32(first), workspace=ws[:size], stream=stream())
    assert bool(torch.isfinite(out.float()).all()) and bool((whole[:3] == 7).all()) and bool((whole[6:] == 7).all()) and bool((ws[size:] == 99).all())


def test_a_cache_beyond_4_gib(attn):
    """Slots and pages whose bytes pass 32 bits."""
    g, kept, dim, n = gen(32), 8, 128, 70000
    pages = torch.empty((n, kept, 72 * dim), dtype=torch.uint8, device="cuda")
    assert pages.numel() > 1 << 32
    cache = attn.Cache(pages, kept, dim)
    used = [n - 1, 3, n - 2, 58254]  # (2^32 bytes lie in the last one)
    slots = torch.cat([torch.arange(p * PAGE, (p + 1) * PAGE) for p in used])[:230].to(torch.int32).cuda()
    k, v = rows(g, 230, kept, dim, "bf16"), rows(g, 230, kept, dim, "bf16")
    attn.store(cache, k, v, slots, stream=stream())
    a, b = torch.empty_like(k), torch.empty_like(v)
    attn.load(cache, slots, a, b, stream=stream())
    assert torch.equal(a, kept64(k).to(torch.bfloat16)) and torch.equal(b, kept64(v).to(torch.bfloat16))
    q, out, table = rows(g, 2, 16, dim, "bf16"), torch.empty((2, 16, dim), dtype=torch.bfloat16, device="cuda"), i32([used])
    attn.attend_cached(cache, q, out, table, i32([230]), i32([0, 2]), workspace=room(attn.attend_cached_workspace(cache, q, table)), stream=stream())
    few = pages[torch.tensor(used, device="cuda")]
    near(out, cached64(q, few, dim, i32([[0, 1, 2, 3]]), [230], [2], dim ** -0.5, 4))


def test_rows_far_apart(attn):
    """Strides whose bytes pass 32 bits: tokens 2^30 + 4 values apart, in every operator that takes rows."""
    g, apart, t, dim = gen(33), (1 << 30) + 4, 3, 64
    flat = torch.empty(2 * apart + 4096, dtype=torch.bfloat16, device="cuda")
    far = lambda at, heads: flat[at:].as_strided((t, heads, dim), (apart, dim, 1))  # noqa: E731
    q, k, v, out = far(0, 4), far(256, 2), far(384, 2), far(512, 4)
    dout, dq, dk, dv = far(768, 4), far(1024, 4), far(1280, 2), far(1408, 2)
    for x in (q, k, v, dout):
        x.copy_(torch.randn(x.shape, device="cuda", generator=g))
    r, positions = attn.Rotary(64), i32([0, 5, 900])
    turned = rotated64(q, positions, r, False)
    attn.rotate(r, positions, q, stream=stream())
    near(q, turned)
    lse = torch.empty((4, t), device="cuda")
    attn.attend(q, k, v, out, lse=lse, stream=stream())
    attn.attend_backward(q, k, v, out, dout, lse, dq, dk, dv, workspace=room(attn.attend_backward_workspace(q, k)), stream=stream())
    want = attend64(q, k, v, [t], [t], True, dim ** -0.5, dout)
    small = BOUND[torch.bfloat16] / 4 * float(dout.double().norm()) * float(v.double().norm(dim=-1).max()) * dim ** -0.5 * 0.05  # (row 0 attends to one key)
    near(out, want[0], "out")
    for name, got, exact in (("dq", dq, want[2]), ("dk", dk, want[3]), ("dv", dv, want[4])):
        near(got, exact, name, slack=0.0 if name == "dv" else small)
    cache = attn.Cache(torch.zeros((1, 2, 72 * dim), dtype=torch.uint8, device="cuda"), 2, dim)
    attn.store(cache, k, v, i32([4, 0, 63]), stream=stream())
    attn.load(cache, i32([4, 0, 63]), dk, dv, stream=stream())
    assert torch.equal(dk, kept64(k).to(torch.bfloat16)) and torch.equal(dv, kept64(v).to(torch.bfloat16))
    attn.attend_cached(cache, q[:1], out[:1], i32([[0]]), i32([1]), i32([0, 1]), workspace=room(attn.attend_cached_workspace(cache, q[:1], i32([[0]]))), stream=stream())
    near(out[:1], kept64(v)[1:2].repeat_interleave(2, 1))


@pytest.mark.parametrize("n", [257, 600])
def test_attend_many_short_sequences(attn, n):
    g, dim = gen(n), 64
    counts = torch.randint(0, 4, (n,), device="cuda", generator=g).tolist()
    counts[n // 2] = 140
    q, k, v, dout, _, first, _ = attend_case("f16", counts, None, 1, 2, dim, "packed", pad=0)
    out, lse = torch.empty_like(q), torch.empty((2, len(q)), device="cuda")
    attn.attend(q, k, v, out, lse=lse, first=first, stream=stream())
    want = attend64(q, k, v, counts, counts, True, dim ** -0.5, dout)
    near(out, want[0])
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    attn.attend_backward(q, k, v, out, dout, lse, dq, dk, dv, first=first, workspace=room(attn.attend_backward_workspace(q, k)), stream=stream())
    for name, got, exact in (("dq", dq, want[2]), ("dk", dk, want[3]), ("dv", dv, want[4])):
        near(got, exact, name)


def test_a_slot_that_is_given_twice_holds_a_mixture_alone(attn):
    """Of values that were given to it, and nothing beside it changes."""
    g = gen(34)
    pages = torch.zeros((2, 2, 72 * 32), dtype=torch.uint8, device="cuda")
    cache, k = attn.Cache(pages, 2, 32), rows(g, 130, 2, 32, "f16")
    slots = torch.full((130,), 70, dtype=torch.int32, device="cuda")
    slots[5] = 3
    attn.store(cache, k, k, slots, stream=stream())
    every = torch.arange(128, device="cuda", dtype=torch.int32)
    a, b = torch.empty((128, 2, 32), dtype=torch.float16, device="cuda"), torch.empty((128, 2, 32), dtype=torch.float16, device="cuda")
    attn.load(cache, every, a, b, stream=stream())
    other = torch.ones(128, dtype=torch.bool, device="cuda")
    other[3] = other[70] = False
    assert bool((a[other] == 0).all()) and bool((b[other] == 0).all())
    assert torch.equal(a[3], kept64(k[5:6]).half()[0]) and bool((a[70].abs() <= k.abs().max()).all())


def test_replays_of_one_operator_each(attn):
    """Captured alone and replayed, with other inputs each time."""
    g = gen(35)
    r, cache = attn.Rotary(64), attn.Cache(random_pages(g, 6, 2, 64), 2, 64)
    positions, k = torch.zeros(70, dtype=torch.int32, device="cuda"), rows(g, 70, 2, 64, "bf16")
    turned, back, back_v = torch.empty_like(k), torch.empty_like(k), torch.empty_like(k)
    at = torch.zeros(70, dtype=torch.int32, device="cuda")
    table, ends, first = i32([[5, 0, 3], [1, 2, 4]]), i32([0, 0]), i32([0, 40, 70])
    q, out = rows(g, 2, 4, 64, "bf16"), torch.empty((2, 4, 64), dtype=torch.bfloat16, device="cuda")
    ws = room(attn.attend_cached_workspace(cache, q, table))
    where = torch.empty(70, dtype=torch.int32, device="cuda")

    def change(i):
        positions.copy_(torch.randint(0, 5000, (70,), device="cuda", generator=g))
        ends.copy_(i32([100 + 13 * i, 64 + 31 * i]))
        k.copy_(torch.randn(k.shape, device="cuda", generator=g))

    def calls():
        attn.rotate(r, positions, k, q_out=turned, stream=stream())
        attn.slots(table, ends, first, where, at, stream=stream())
        attn.store(cache, turned, k, at, stream=stream())
        attn.load(cache, at, back, back_v, stream=stream())
        attn.attend_cached(cache, q, out, table, ends, i32_one, workspace=ws, stream=stream())

    i32_one = i32([0, 1, 2])
    change(0)
    state = {"i": 0}

    def check(_):
        near(turned, rotated64(k, positions, r, False))
        assert torch.equal(back, kept64(turned).to(torch.bfloat16)) and torch.equal(back_v, kept64(k).to(torch.bfloat16))
        near(out, cached64(q, cache.pages, 64, table, ends.tolist(), [1, 1], 0.125, 6))
        state["i"] += 1
        change(state["i"])

    replays(calls, check)
