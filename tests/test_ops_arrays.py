"""What tierstream_amd.ops refuses of the arrays it is given, before their addresses reach the library: no GPU is needed."""
import pytest

from tierstream_amd import ops
from test_ops_refusals import Fake, experts


class Array(Fake):
    """A contiguous array of any number of axes."""

    def __init__(self, *shape, dtype="torch.bfloat16"):
        stride = [1]
        for n in shape[:0:-1]:
            stride.insert(0, stride[0] * n)
        super().__init__(*shape, dtype=dtype, stride=tuple(stride))

    def is_contiguous(self):
        return True


class Host(Array):
    is_cuda = False


def holder():
    e = ops.Experts(1, 64, 96, "bf16")
    e.s = experts()
    return e


def i32(cls, *shape):
    return cls(*shape, dtype="torch.int32")


def f32(cls, *shape):
    return cls(*shape, dtype="torch.float32")


CALLS = {
    "logits": lambda h: ops.route(f32(h["logits"], 2, 64), i32(Fake, 2, 8), f32(Fake, 2, 8)),
    "ids": lambda h: ops.route(f32(Fake, 2, 64), i32(h["ids"], 2, 8), f32(Fake, 2, 8)),
    "dlogits": lambda h: ops.route_backward(f32(Fake, 2, 64), i32(Fake, 2, 8), f32(Fake, 2, 8), f32(h["dlogits"], 2, 64)),
    "x": lambda h: ops.linear(h["x"](2, 128), Fake(64, 128), Fake(2, 64)),
    "w": lambda h: ops.linear(Fake(2, 128), h["w"](64, 128), Fake(2, 64)),
    "y": lambda h: ops.linear(Fake(2, 128), Fake(64, 128), h["y"](2, 64)),
    "bias": lambda h: ops.linear(Fake(2, 128), Fake(64, 128), Fake(2, 64), bias=h["bias"](64)),
    "residual": lambda h: ops.linear(Fake(2, 128), Fake(64, 128), Fake(2, 64), residual=h["residual"](2, 64)),
    "workspace": lambda h: ops.ffn(holder(), Fake(2, 64), Fake(2, 64), ids=i32(Fake, 2, 2), workspace=h["workspace"](1, 64)),
    "weights": lambda h: ops.ffn(holder(), Fake(2, 64), Fake(2, 64), ids=i32(Fake, 2, 2), weights=f32(h["weights"], 2, 2)),
    "dy": lambda h: ops.ffn_backward(holder(), Fake(2, 64), h["dy"](2, 64), ids=i32(Fake, 2, 2)),
    "gate": lambda h: ops.Experts.stacked(h["gate"](2, 96, 64), Array(2, 96, 64), Array(2, 64, 96)),
    "table": lambda h: ops.Experts.in_table(h["table"](4, dtype="torch.int64"), 64, 96, "bf16"),
}


@pytest.mark.parametrize("name", CALLS)
def test_an_array_of_the_host_is_refused(name):
    with pytest.raises(ValueError, match=f"{name}.*device memory"):
        CALLS[name]({name: Host})


class Spaced(Array):
    def is_contiguous(self):
        return False


@pytest.mark.parametrize("table", [Array(8, dtype="torch.int32"), Array(4, dtype="torch.float64"), Array(2, 4, dtype="torch.int64"),
                                   Spaced(4, dtype="torch.int64")])
def test_a_table_is_an_array_of_64_bit_addresses(table):
    with pytest.raises(ValueError, match="table"):
        ops.Experts.in_table(table, 64, 96, "bf16")
    assert ops.Experts.in_table(Array(4, dtype="torch.int64"), 64, 96, "bf16").s.table


@pytest.mark.parametrize("f,width,wide", [(96, 37, 54), (96, 17, 54), (80, 36, 36)])
def test_stacked_4_bit_rows_are_whole_blocks(f, width, wide):
    parts = [Array(2, f, width, dtype="torch.uint8"), Array(2, f, width, dtype="torch.uint8"), Array(2, width // 18 * 32, wide, dtype="torch.uint8")]
    with pytest.raises(ValueError, match="blocks"):
        ops.Experts.stacked(*parts)
