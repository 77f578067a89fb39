"""Scores of attention over the 4-bit cache on an MI355X, where they are large and far apart from 0: what 32 bits lose of them goes to the
probabilities as it is."""
import gc

import pytest
import torch

from test_gpu_ops_attn import KINDS, PAGE, gen, i32, numbers64, room, stream

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def attn(gpu):
    from tierstream_amd import attn
    yield attn
    gc.collect()
    torch.cuda.synchronize()


def put(pages, dim, at, part, whole, scale):
    """Whole numbers -8..7 [dim], times scale, as the key (0) or value (1) of slot `at`."""
    page, token, nb = pages[at // PAGE, 0], at % PAGE, dim // 32
    b = (whole.view(nb, 32) + 8).to(torch.uint8)
    packed = b[:, :16] | b[:, 16:] << 4
    if part:
        page[40 * dim:].view(nb, PAGE, 16)[:, token] = packed
    else:
        page[:32 * dim].view(PAGE, 4, nb, 4)[token] = packed.view(nb, 4, 4).transpose(0, 1)
    page[(32 + 4 * part) * dim:(36 + 4 * part) * dim].view(torch.float16).view(PAGE, nb)[token] = scale


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("a,b", [(0, 1), (5, 62), (3, 70), (130, 20)])
def test_equal_scores_share_alike(attn, kind, dim, a, b):
    """Queries above 0 whose values come in equal pairs, anywhere in a head, and two keys that differ by the order of each pair: their scores, some hundred, are the same number, a
    whole number of some unit. A query has 11 bits (8), a kept number 4, the sum over a head 7 more: below 2^24 units, so that sums in 32 bits of
    products with the kept numbers, or with numbers a few times as large, are exact. Both probabilities are 1/2 then, and the output is half the values' sum,
    which 16 bits hold. Every other key scores 0."""
    g, heads = gen(dim + a), 16
    pages = torch.zeros((3, 1, 72 * dim), dtype=torch.uint8, device="cuda")
    for at in range(3 * PAGE):
        put(pages, dim, at, 0, torch.zeros(dim, dtype=torch.int64, device="cuda"), 1.0)
        put(pages, dim, at, 1, torch.randint(-8, 8, (dim,), device="cuda", generator=g), 0.5)
    bits = 11 if kind == "f16" else 8
    pairs = torch.randint(1 << (bits - 1), 1 << bits, (heads, dim // 2), device="cuda", generator=g).double()
    where = torch.argsort(torch.randperm(dim, device="cuda", generator=g))
    q = (pairs * 2.0 ** (2 - bits)).repeat_interleave(2, 1)[:, where][None].to(KINDS[kind])
    one = torch.randint(1, 8, (dim // 2, 2), device="cuda", generator=g)
    put(pages, dim, a, 0, one.flatten()[where], 32.0)
    put(pages, dim, b, 0, one.flip(1).flatten()[where], 32.0)
    keys, values = numbers64(pages, dim)[:, :, 0].reshape(2, -1, dim)
    scores = q[0].double() @ keys.T
    assert torch.equal(scores[:, a], scores[:, b]) and float(scores[:, a].min()) * dim ** -0.5 > 200
    cache, table, out = attn.Cache(pages, 1, dim), i32([[0, 1, 2]]), torch.empty_like(q)
    attn.attend_cached(cache, q, out, table, i32([3 * PAGE]), i32([0, 1]), workspace=room(attn.attend_cached_workspace(cache, q, table)), stream=stream())
    assert torch.equal(out[0].double(), ((values[a] + values[b]) / 2).expand(heads, dim))
