"""The attention operators on an MI355X where their documents allow more than a step needs: lists that do not begin at the first row, or whose
spans overlap by far; nothing out of range is read or written, and rows that no request or sequence has are left as they were."""
import gc

import pytest
import torch

from test_gpu_ops_attn import i32, stream

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def attn(gpu):
    from tierstream_amd import attn
    yield attn
    gc.collect()
    torch.cuda.synchronize()


def test_rows_before_the_first_request_have_no_slot(attn):
    """Request i has the rows first[i]..first[i + 1]: those before first[0] belong to none, and a store to their slots would overwrite older
    tokens of the first request."""
    positions, slots = i32([9] * 10), i32([9] * 10)
    attn.slots(i32([[1, 2], [4, 0]]), i32([100, 3]), i32([3, 5, 8]), positions, slots, stream=stream())
    assert positions.tolist() == [-1] * 3 + [98, 99, 0, 1, 2] + [-1] * 2
    assert slots.tolist() == [-1] * 3 + [162, 163, 256, 257, 258] + [-1] * 2
    attn.slots(i32([[1, 2]]), i32([70]), i32([12, 20]), positions, slots, stream=stream())  # (all of them)
    assert positions.tolist() == [-1] * 10 and slots.tolist() == [-1] * 10


def test_requests_that_overlap_beyond_all_counts(attn):
    """4096 requests that each say to have all of 16384 tokens, or none: 2048 x 16384 tiles x 255 rounds, more than 32 bits count."""
    tokens, requests, width, dim = 16384, 4096, 1020, 32
    cache = attn.Cache(torch.zeros((4, 1, 72 * dim), dtype=torch.uint8, device="cuda"), 1, dim)
    table = torch.arange(requests * width, device="cuda", dtype=torch.int32).view(requests, width) % 4
    whole = torch.full((tokens + 2, 16, dim), 7.0, dtype=torch.float16, device="cuda")
    q, out = torch.ones((tokens, 16, dim), dtype=torch.float16, device="cuda"), whole[1:-1]
    size = attn.attend_cached_workspace(cache, q, table)
    ws = torch.full((size + 1024,), 99, dtype=torch.uint8, device="cuda")
    ends = torch.full((requests,), width * 64, dtype=torch.int32, device="cuda")
    attn.attend_cached(cache, q, out, table, ends, i32([0, tokens] * (requests // 2) + [0]), workspace=ws[:size], stream=stream())
    torch.cuda.synchronize()
    assert bool((whole[0] == 7).all()) and bool((whole[-1] == 7).all()) and bool((ws[size:] == 99).all())
    attn.attend_cached(cache, q[:2], out[:2], table[:2], ends[:2], i32([0, 1, 2]), workspace=ws[:size], stream=stream())
    assert bool((out[:2] == 0).all())  # (pages of zeros)


def test_sequences_that_overlap_beyond_all_counts(attn):
    """65536 sequences that each say to have all of 2^24 - 1 rows, or none: 32768 x 131072 tiles are 2^32. None is taken up; then two that
    follow each other are."""
    many, few, n = (1 << 24) - 1, 16, 1 << 16
    wide, small = torch.ones((many, 1, 8), dtype=torch.bfloat16, device="cuda"), torch.ones((few, 1, 8), dtype=torch.bfloat16, device="cuda")
    far, near = i32([0, many] * (n // 2) + [0]), i32([0] * n + [few])
    out, lse = torch.full_like(wide, 7.0), torch.full((1, many), 7.0, device="cuda")
    ws = torch.empty(attn.attend_backward_workspace(wide, small), dtype=torch.uint8, device="cuda")
    attn.attend(wide, small, small, out, lse=lse, first=far, k_first=near, stream=stream())
    assert bool((out == 7).all()) and bool((lse == 7).all())
    dq = torch.full_like(wide, 7.0)
    attn.attend_backward(wide, small, small, out, wide, lse, dq, first=far, k_first=near, workspace=ws, stream=stream())
    assert bool((dq == 7).all())
    out[:20], lse[:, :20] = 7.0, 7.0
    attn.attend(wide, small, small, out, lse=lse, first=i32([0, 9, 20]), k_first=i32([0, 9, 16]), causal=False, stream=stream())
    assert bool((out[:20] == 1).all()) and bool((out[20:] == 7).all())
    del out, lse, dq
    ws = torch.empty(attn.attend_backward_workspace(small, wide), dtype=torch.uint8, device="cuda")
    dk, dv, out, lse = torch.full_like(wide, 7.0), torch.full_like(wide, 7.0), torch.ones_like(small), torch.zeros((1, few), device="cuda")
    attn.attend_backward(small, wide, wide, out, small, lse, None, dk, dv, first=near, k_first=far, workspace=ws, stream=stream())
    assert bool((dk == 7).all()) and bool((dv == 7).all())
