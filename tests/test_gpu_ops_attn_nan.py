"""Where infinities and NaN of the attention operators' inputs go on an MI355X: into every row that attends to them, and into no other. One
value at a time, in each part of a workgroup's tile of 128 own rows and of the tiles of 64 that it runs over: what a mask takes out of a tile
for some of the waves, the others have to see."""
import gc
import math

import pytest
import torch

from test_gpu_ops_attn import attend_case, room, stream

pytestmark = pytest.mark.gpu

CASES = [  # queries, keys (None: as many), dim: sequences of one row, of parts of tiles, of whole ones, with more keys than queries and with fewer
    ([100], None, 64), ([256], None, 128), ([1, 200, 70], None, 72), ([130], [333], 64), ([300], [210], 128)]


@pytest.fixture(scope="module")
def attn(gpu):
    from tierstream_amd import attn
    yield attn
    gc.collect()
    torch.cuda.synchronize()


def attended(counts, k_counts):
    """[queries][keys]: which query attends to which key, under a causal mask."""
    ok = torch.zeros((sum(counts), sum(k_counts)), dtype=torch.bool, device="cuda")
    a = b = 0
    for n, m in zip(counts, k_counts):
        ok[a:a + n, b:b + m] = torch.ones((n, m), dtype=torch.bool, device="cuda").tril(m - n)
        a, b = a + n, b + m
    return ok


def places(n):
    """Rows of n in every quarter of a tile of 128, at both ends of each."""
    return sorted({i for i in (0, 5, 31, 32, 63, 64, 70, 95, 96, 127, 128, 150, 191, 192, 209, 255, n - 1) if i < n})


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("counts,k_counts,dim", CASES)
@pytest.mark.parametrize("layout", ["packed", "odd"])
def test_a_value_that_is_no_number(attn, kind, counts, k_counts, dim, layout):
    """In V: every output of a row that attends to it has none in its place, and all others are as with a 0 there."""
    q, k, v, _, k_counts, first, k_first = attend_case(kind, counts, k_counts, 2, 2, dim, layout, pad=0)
    ok, where = attended(counts, k_counts), dict(first=first, k_first=k_first, stream=stream())
    lse, out, plain = torch.empty((4, len(q)), device="cuda"), torch.empty_like(q), torch.empty_like(q)
    for i, j in enumerate(places(len(v))):
        d, was = (7 * j) % dim, v[j, 1, (7 * j) % dim].clone()
        v[j, 1, d] = 0
        attn.attend(q, k, v, plain, lse=lse, **where)
        v[j, 1, d] = (math.nan, math.inf, -math.inf)[i % 3]
        attn.attend(q, k, v, out, lse=lse, **where)
        v[j, 1, d] = was
        sees = ok[:, j]
        assert not bool(torch.isfinite(out[sees][:, 2:, d].float()).any()), f"key {j}: lost"
        assert torch.equal(out[~sees], plain[~sees]) and torch.equal(out[:, :2], plain[:, :2]), f"key {j}: elsewhere"


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("counts,k_counts,dim", CASES)
def test_a_key_or_a_query_that_is_no_number(attn, kind, counts, k_counts, dim):
    """A key's: outputs and log sums of the rows that attend to it. A query's: its own row's."""
    q, k, v, _, k_counts, first, k_first = attend_case(kind, counts, k_counts, 2, 2, dim, "packed", pad=0)
    ok, where = attended(counts, k_counts), dict(first=first, k_first=k_first, stream=stream())
    one, lse, out, plain = torch.empty((4, len(q)), device="cuda"), torch.empty((4, len(q)), device="cuda"), torch.empty_like(q), torch.empty_like(q)
    attn.attend(q, k, v, plain, lse=one, **where)
    for x, at in ((k, places(len(k))), (q, places(len(q)))):
        for j in at:
            head, was = len(x[j]) - 1, x[j, -1, 3].clone()
            x[j, head, 3] = math.nan
            attn.attend(q, k, v, out, lse=lse, **where)
            x[j, head, 3] = was
            bad = torch.zeros((len(q), 4), dtype=torch.bool, device="cuda")
            if x is k:
                bad[:, 2:] = ok[:, j:j + 1]
            else:
                bad[j, 3] = bool(ok[j].any())  # (a row without keys is 0)
            assert bool(out[bad].isnan().all()) and bool(lse.T[bad].isnan().all()), f"{'key' if x is k else 'query'} {j}: lost"
            if x is q:
                assert torch.equal(out[~bad], plain[~bad]) and torch.equal(lse.T[~bad], one.T[~bad]), f"query {j}: elsewhere"
            else:
                assert torch.equal(out[:, :2], plain[:, :2]) and bool(torch.isfinite(out[~bad].float()).all()), f"key {j}: elsewhere"


def gradients(attn, q, k, v, dout, where):
    out, lse = torch.empty_like(q), torch.empty((q.shape[1], len(q)), device="cuda")
    attn.attend(q, k, v, out, lse=lse, **where)
    grads = [torch.full_like(x, 7.0) for x in (q, k, v)]
    attn.attend_backward(q, k, v, out, dout, lse, *grads, workspace=room(attn.attend_backward_workspace(q, k)), **where)
    return out, lse, grads


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("counts,k_counts,dim", CASES)
@pytest.mark.parametrize("layout", ["packed", "odd"])
def test_queries_gradients_with_a_key_of_no_score(attn, kind, counts, k_counts, dim, layout):
    """A key's value of -infinity where queries are positive: its probability is 0 and outputs are numbers, but dq = sum ds k has 0 x infinity
    in that value for every row that attends to it. Rows that do not are as with a 0 there."""
    q, k, v, dout, k_counts, first, k_first = attend_case(kind, counts, k_counts, 2, 2, dim, layout, pad=0)
    ok, where = attended(counts, k_counts), dict(first=first, k_first=k_first, stream=stream())
    for j in places(len(k)):
        d = (5 * j) % dim
        had, was = q[:, :, d].clone(), k[j, 1, d].clone()
        q[:, :, d] = 1
        k[j, 1, d] = 0
        _, _, plain = gradients(attn, q, k, v, dout, where)
        k[j, 1, d] = -math.inf
        out, _, got = gradients(attn, q, k, v, dout, where)
        q[:, :, d], k[j, 1, d] = had, was
        sees = ok[:, j]
        assert bool(torch.isfinite(out.float()).all())
        assert bool(got[0][sees][:, 2:, d].isnan().all()), f"key {j}: lost"
        assert torch.equal(got[0][~sees], plain[0][~sees]) and torch.equal(got[0][:, :2], plain[0][:, :2]), f"key {j}: elsewhere"


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("counts,k_counts,dim", CASES)
@pytest.mark.parametrize("layout", ["packed", "odd"])
def test_keys_gradients_with_a_row_that_is_no_number(attn, kind, counts, k_counts, dim, layout):
    """One value of dout, or of a query: the gradients of every key that its row attends to, of its own query, and of no other."""
    q, k, v, dout, k_counts, first, k_first = attend_case(kind, counts, k_counts, 2, 2, dim, layout, pad=0)
    ok, where = attended(counts, k_counts), dict(first=first, k_first=k_first, stream=stream())
    for x in (dout, q):
        for i, row in enumerate(places(len(q))):
            d, was = (3 * row) % dim, x[row, 2, (3 * row) % dim].clone()
            x[row, 2, d] = 0
            _, _, plain = gradients(attn, q, k, v, dout, where)
            x[row, 2, d] = (math.nan, math.inf, -math.inf)[i % 3] if x is dout else math.nan
            _, _, (dq, dk, dv) = gradients(attn, q, k, v, dout, where)
            x[row, 2, d] = was
            seen, own = ok[row], torch.zeros((len(q), 4), dtype=torch.bool, device="cuda")
            own[row, 2] = bool(seen.any())
            what = f"{'dout' if x is dout else 'query'} {row}"
            assert not bool(torch.isfinite(dv[seen][:, 1, d if x is dout else slice(None)].float()).any()), f"{what}: lost in dv"
            assert not bool(torch.isfinite(dk[seen][:, 1].float()).any()), f"{what}: lost in dk"
            assert not bool(torch.isfinite(dq[own].float()).any()), f"{what}: lost in dq"
            for got, want in ((dk, plain[1]), (dv, plain[2])):
                assert torch.equal(got[~seen], want[~seen]) and torch.equal(got[:, 0], want[:, 0]), f"{what}: elsewhere"
            assert torch.equal(dq[~own], plain[0][~own]), f"{what}: elsewhere in dq"


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("counts,k_counts,dim", CASES)
def test_gradients_with_a_value_that_is_no_number(attn, kind, counts, k_counts, dim):
    """In V: dq of every row that attends to it, and dk of every key that such a row attends to."""
    q, k, v, dout, k_counts, first, k_first = attend_case(kind, counts, k_counts, 2, 2, dim, "packed", pad=0)
    ok, where = attended(counts, k_counts), dict(first=first, k_first=k_first, stream=stream())
    for j in places(len(v)):
        was = v[j, 1, 1].clone()
        v[j, 1, 1] = math.nan
        _, _, (dq, dk, _) = gradients(attn, q, k, v, dout, where)
        v[j, 1, 1] = was
        sees = ok[:, j]
        met = ok[sees].any(0)
        assert not bool(torch.isfinite(dq[sees][:, 2:].float()).any()) and not bool(torch.isfinite(dk[met][:, 1].float()).any()), f"key {j}: lost"
        assert bool(torch.isfinite(dq[~sees].float()).all()) and bool(torch.isfinite(dk[~met].float()).all()), f"key {j}: elsewhere"
        assert bool(torch.isfinite(dq[:, :2].float()).all()) and bool(torch.isfinite(dk[:, 0].float()).all()), f"key {j}: elsewhere"
