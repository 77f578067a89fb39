"""Paths of the attention operators on an MI355X that few shapes take: keys' gradients of calls with many heads, which are cut into few pieces or
none; scales of the cache that are no numbers among a request's new tokens; and what lies between rows that are turned in place."""
import gc
import math

import pytest
import torch

from test_gpu_ops_attn import KINDS, PAGE, attend64, cached64, first_of, gen, i32, near, random_pages, rotated64, room, rows, stream

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def attn(gpu):
    from tierstream_amd import attn
    yield attn
    gc.collect()
    torch.cuda.synchronize()


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("layout", ["packed", "odd"])
@pytest.mark.parametrize("counts,kept,group,dim", [  # (rows / 128 + 1) x kept heads: from 1024 on keys' queries are in one piece, down to 147 in up to 7
    ([40], 1024, 1, 64), ([23, 17], 1024, 1, 72), ([40], 1024, 1, 128), ([200, 100], 512, 2, 64), ([40], 520, 1, 128), ([100], 400, 2, 72), ([30], 300, 1, 64),
    ([70], 150, 1, 128), ([400], 256, 1, 64), ([20, 400], 256, 1, 128)])
def test_gradients_of_many_heads(attn, kind, layout, counts, kept, group, dim):
    g, t = gen(sum(counts) + kept), sum(counts)
    q, dout = rows(g, t, kept * group, dim, kind, layout), rows(g, t, kept * group, dim, kind, layout, 0.1)
    k, v = rows(g, t, kept, dim, kind, layout), rows(g, t, kept, dim, kind, layout)
    new = lambda x: rows(None, *x.shape, kind, layout, fill=7.0)  # noqa: E731
    out, lse, dq, dk, dv = new(q), torch.empty((kept * group, t), device="cuda"), new(q), new(k), new(v)
    size, where = attn.attend_backward_workspace(q, k), dict(first=first_of(counts), stream=stream())
    ws = torch.full((size + 4096,), 99, dtype=torch.uint8, device="cuda")
    attn.attend(q, k, v, out, lse=lse, **where)
    attn.attend_backward(q, k, v, out, dout, lse, dq, dk, dv, workspace=ws[:size], **where)
    want = attend64(q, k, v, counts, counts, True, dim ** -0.5, dout)
    near(out, want[0], "out")
    for name, got, exact in (("dq", dq, want[2]), ("dk", dk, want[3]), ("dv", dv, want[4])):
        near(got, exact, name)
    assert bool((ws[size:] == 99).all())
    again = new(k), new(v)
    attn.attend_backward(q, k, v, out, dout, lse, None, *again, workspace=ws[:size], **where)
    assert torch.equal(again[0], dk) and torch.equal(again[1], dv)


def scales_of(pages, dim, part):
    """[n][kept][64 tokens][blocks] of keys (0) or values (1), in place."""
    at = (32 + 4 * part) * dim
    return pages[..., at:at + 4 * dim].view(torch.float16).view(*pages.shape[:2], PAGE, dim // 32)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("end,fresh", [(200, 3), (193, 3), (192, 5), (66, 66), (700, 20)])
def test_scales_that_are_no_numbers(attn, kind, dim, end, fresh):
    """Of one block of a value or a key: rows that attend to it have none in its place (a key: in any), all others are as with a scale of 0."""
    g, n, kept, group = gen(end + dim), (end + PAGE - 1) // PAGE, 2, 3
    pages, table = random_pages(g, n, kept, dim), torch.arange(n, device="cuda", dtype=torch.int32)[None]
    cache, q = attn.Cache(pages, kept, dim), rows(g, fresh, kept * group, dim, kind)
    size = attn.attend_cached_workspace(cache, q, table)
    ws, out, plain = torch.empty(size, dtype=torch.uint8, device="cuda"), torch.empty_like(q), torch.empty_like(q)
    call = lambda y: attn.attend_cached(cache, q, y, table, i32([end]), i32([0, fresh]), workspace=ws, stream=stream())  # noqa: E731
    places = sorted({0, 63, 64, end - fresh - 1, end - fresh, end - fresh + 1, end - 2, end - 1} & set(range(end)))
    for part in (1, 0):
        scales = scales_of(pages, dim, part)
        for i, j in enumerate(places):
            block = i % (dim // 32)
            at = scales[j // PAGE, 1, j % PAGE]
            was = at[block].clone()
            at[block] = 0
            call(plain)
            at[block] = (math.nan, math.inf, -math.inf)[i % 3] if part else math.nan
            call(out)
            at[block] = was
            sees = torch.arange(end - fresh, end, device="cuda") >= j
            what = f"{'value' if part else 'key'} {j}"
            bad = out[sees][:, group:]
            assert not bool(torch.isfinite((bad[..., 32 * block:32 * block + 32] if part else bad).float()).any()), f"{what}: lost"
            assert torch.equal(out[~sees], plain[~sees]) and torch.equal(out[:, :group], plain[:, :group]), f"{what}: elsewhere"


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,kept,dim,rotated,layout", [(700, 8, 2, 128, 64, "slice"), (33, 5, 1, 72, 18, "odd"), (4, 32, 8, 128, 128, "packed")])
def test_turned_in_place(attn, kind, interleaved, tokens, heads, kept, dim, rotated, layout):
    """Queries and keys together, there and back: what lies between and behind their rows stays, and so does what is turned elsewhere."""
    g, r = gen(tokens + dim), attn.Rotary(rotated, interleaved=interleaved, amplitude=1.1)
    pad, shift = {"packed": (0, 0), "slice": (16, 8), "odd": (3, 1)}[layout]
    width = (heads + kept) * dim + pad
    flat = torch.randn(tokens * width + shift + 8, device="cuda", generator=g).to(KINDS[kind])
    x = flat[shift:].as_strided((tokens, heads + kept, dim), (width, dim, 1))
    positions = torch.randint(0, 4096, (tokens,), device="cuda", generator=g, dtype=torch.int32)
    positions[tokens // 2] = -1
    live = positions >= 0
    for backward in (False, True):
        before, want = flat.clone(), rotated64(x, positions, r, backward)
        out = torch.empty_like(x), torch.empty_like(x)
        attn.rotate(r, positions, x[:, :heads], x[:, heads:], out[0][:, :heads], out[1][:, heads:], backward=backward, stream=stream())
        assert torch.equal(flat, before)
        attn.rotate(r, positions, x[:, :heads], x[:, heads:], backward=backward, stream=stream())
        near(x[live], want[live])
        assert torch.equal(x[live][:, :heads], out[0][live][:, :heads]) and torch.equal(x[live][:, heads:], out[1][live][:, heads:])
        inside = torch.zeros(len(flat), dtype=torch.bool, device="cuda")
        inside[shift:].as_strided((tokens, heads + kept, dim), (width, dim, 1))[live] = True
        assert torch.equal(flat[~inside], before[~inside])


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("ends,fresh,kept,group,dim", [([1500, 700], [1000, 300], 1, 4, 64), ([600, 64, 900], [600, 1, 33], 2, 3, 128), ([2000], [250], 2, 8, 96)])
def test_chunks_of_a_prompt_over_the_cache(attn, kind, ends, fresh, kept, group, dim):
    """Hundreds of new tokens a request, from the first one on or behind a long context: tiles of 16 rows that begin and end inside tokens."""
    g, tokens = gen(sum(ends)), sum(fresh)
    need = [(e + PAGE - 1) // PAGE for e in ends]
    pages, table = random_pages(g, sum(need), kept, dim), torch.full((len(ends), max(need)), -1, dtype=torch.int32, device="cuda")
    order = torch.randperm(sum(need), device="cuda", generator=g).to(torch.int32)
    for i, n in enumerate(need):
        table[i, :n] = order[sum(need[:i]):sum(need[:i]) + n]
    q, out, cache = rows(g, tokens, kept * group, dim, kind), rows(g, tokens, kept * group, dim, kind, fill=7.0), attn.Cache(pages, kept, dim)
    attn.attend_cached(cache, q, out, table, i32(ends), first_of(fresh), workspace=room(attn.attend_cached_workspace(cache, q, table)), stream=stream())
    near(out, cached64(q, pages, dim, table, ends, fresh, dim ** -0.5, len(pages)))
