"""Attention over packed sequences on an MI355X: what a sequence's results do not depend on (what else is in the call, where it lies in memory).

Outputs, log sums and queries' gradients are made by workgroups of one sequence: the same bits. Sums of keys' gradients are cut by how many keys
the call has, in 32 bits: off by about sqrt(300) 2^-24 of the terms, by which one value in 2000 (bf16) or 250 (half precision) rounds to its neighbour,
2^-8 or 2^-11 away: 1e-4 or 3e-5 in the 2-norm. Four times that is allowed; probabilities rounded once more or less would be 1.6e-3 or 2e-4."""
import gc

import pytest
import torch

from test_gpu_ops_attn import KINDS, attend64, first_of, gen, room, rows, stream

pytestmark = pytest.mark.gpu

SAME = {torch.bfloat16: 4e-4, torch.float16: 1.2e-4}


@pytest.fixture(scope="module")
def attn(gpu):
    from tierstream_amd import attn
    yield attn
    gc.collect()
    torch.cuda.synchronize()


def both(attn, q, k, v, dout, counts, causal, layout="packed"):
    kind = {v: k for k, v in KINDS.items()}[q.dtype]
    at = lambda x: rows(None, *x.shape, kind, layout, fill=7.0).copy_(x)  # noqa: E731
    q, k, v, dout = at(q), at(k), at(v), at(dout)
    out, lse, grads = at(q), torch.empty((q.shape[1], len(q)), device="cuda"), [at(x) for x in (q, k, v)]
    where = dict(first=first_of(counts), causal=causal, stream=stream())
    attn.attend(q, k, v, out, lse=lse, **where)
    attn.attend_backward(q, k, v, out, dout, lse, *grads, workspace=room(attn.attend_backward_workspace(q, k)), **where)
    return out, lse.T, *grads


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n,others", [(301, [700, 33]), (100, [1] * 30 + [400]), (700, [50, 60])])
def test_a_sequence_is_the_same_in_any_batch(attn, kind, dim, n, others):
    """Alone, and behind or before others; beside aligned rows, and at odd places."""
    g, counts = gen(n + dim), [*others, n, *others]
    at = sum(others)
    q, k, v, dout = (rows(g, sum(counts), h, dim, kind) for h in (4, 2, 2, 4))
    own = [x[at:at + n] for x in (q, k, v, dout)]
    alone = both(attn, *own, [n], True)
    for got in ([x[at:at + n] for x in both(attn, q, k, v, dout, counts, True)], both(attn, *own, [n], True, "odd")):
        for name, x, y in zip(("out", "lse", "dq"), got, alone):
            assert torch.equal(x, y), name
        for name, x, y in zip(("dk", "dv"), got[3:], alone[3:]):
            assert float((x.double() - y.double()).norm()) <= SAME[x.dtype] * float(y.double().norm()), name


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_short_sequences_are_as_exact_as_their_results(attn, kind):
    """Of at most 2^17 pairs: what rounding probabilities and scores' gradients leaves is multiplied too, so that the rounding of the results is
    what is left. Its mean square over the values is (half a step)^2 / 3 at the lower end of a binade and a quarter of that at the upper one:
    0.737 of half a step / sqrt(3) for normal values. A tenth more is allowed for sums in 32 bits; one more rounding would be sqrt(2) of it."""
    g, dim, counts = gen(5), 64, [300, 361, 20]
    q, k, v, dout = (rows(g, sum(counts), h, dim, kind) for h in (8, 2, 2, 8))
    got = both(attn, q, k, v, dout, counts, True)
    want = attend64(q, k, v, counts, counts, True, dim ** -0.5, dout)
    bound = 1.1 * 0.737 * torch.finfo(q.dtype).eps / 2 / 3 ** 0.5
    for name, x, y in zip(("out", "dq", "dk", "dv"), (got[0], *got[2:]), (want[0], *want[2:])):
        assert float((x.double() - y).norm()) <= bound * float(y.norm()), name
