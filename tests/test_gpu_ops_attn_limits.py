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
