"""What the model operators refuse (include/tierstream_amd/tsa_ops.h), before any launch: no GPU is needed."""
import ctypes as C
from pathlib import Path

import pytest

import tierstream_amd as tsa
from test_abi import declared
from tierstream_amd import ops, ss

ROOT = Path(__file__).resolve().parent.parent
P = 0x10000  # an address that is never read


def refused(call, *args, status=tsa.SS_E_INVALID, says=""):
    got = call(*args)
    msg = tsa.lib().ss_last_error().decode()
    assert got == status, (got, msg)
    assert says in msg, msg


def changed(struct, **fields):
    c = type(struct)()
    C.memmove(C.addressof(c), C.addressof(struct), C.sizeof(c))
    for k, v in fields.items():
        setattr(c, k, v)
    return c


def test_every_declared_operator_is_exported():
    names = declared(ROOT / "include" / "tierstream_amd" / "tsa_ops.h")
    assert len(names) == 8
    assert [n for n in names if not hasattr(tsa.lib(), n)] == []


def test_route():
    f = ops._ops().tsa_route
    a = ops.TsaRouteArgs(logits=P, logits_stride=64, ids=P, weights=P, rows=4, n_experts=64, top_k=8, type=ops.F32, renorm=1, scale=1)
    refused(f, None, None, says="null")
    for bad in (dict(n_experts=0), dict(n_experts=1025), dict(top_k=0), dict(top_k=65), dict(n_experts=4, top_k=5), dict(type=ops.Q4),
                dict(renorm=2), dict(scale=float("nan")), dict(logits=None), dict(logits=P + 2), dict(logits_stride=63), dict(ids=None),
                dict(weights=P + 1)):
        refused(f, C.byref(changed(a, **bad)), None, says="tsa_route")
    b = ops._ops().tsa_route_backward
    refused(b, C.byref(a), None, P, 64, None, says="dweights")
    refused(b, C.byref(a), P, None, 64, None, says="dlogits")
    refused(b, C.byref(a), P, P, 10, None, says="dlogits")
    assert f(C.byref(changed(a, rows=0, logits=None)), None) == tsa.SS_OK


def test_linear():
    f = ops._ops().tsa_linear
    a = ops.TsaLinearArgs(x=P, x_stride=128, w=P, w_stride=128, y=P, y_stride=64, rows=2, n_in=128, n_out=64, x_type=ops.BF16,
                          w_type=ops.BF16, y_type=ops.BF16, act=0)
    refused(f, None, None, 0, None)
    for bad in (dict(x_type=ops.F32), dict(w_type=ops.F16), dict(y_type=ops.F16), dict(act=5), dict(n_in=0), dict(x=None),
                dict(x=P + 1), dict(x_stride=127), dict(w=None), dict(w_stride=100), dict(y=None), dict(y_stride=63),
                dict(y_type=ops.F32, y=P + 2), dict(residual=P, residual_stride=3), dict(bias=P + 1), dict(rows=1 << 31),
                dict(w_type=ops.Q4, n_in=120), dict(w_type=ops.Q4, w_stride=256), dict(w_type=ops.Q4, w=P + 2)):
        refused(f, C.byref(changed(a, **bad)), P, 1 << 40, None, says="tsa_linear")
    refused(f, C.byref(a), P + 8, 1 << 40, None, says="workspace")
    assert f(C.byref(changed(a, rows=0, x=None)), None, 0, None) == tsa.SS_OK


def experts(**kw):
    e = ops.TsaExperts(n_experts=4, d_model=64, d_ff=96, w_type=ops.BF16)
    for p in range(3):
        e.part[p], e.part_stride[p] = P, 64 * 96 * 2
    for k, v in kw.items():
        setattr(e, k, v)
    return e


def view(**kw):
    v = ss.SsDgDeviceView(struct_size=C.sizeof(ss.SsDgDeviceView), n_gated=2, n_parts=3, guard_slot=3, slots=4, slot_of=P, unit_base=P,
                          abort=P)
    for p in range(3):
        v.parts[p].base, v.parts[p].stride, v.parts[p].bytes = P, 64 * 96 * 2, 64 * 96 * 2
    for k, w in kw.items():
        setattr(v, k, w)
    return v


def bad_experts():
    none = experts()
    none.part[0] = None
    two = experts(table=P)
    part = experts()
    part.part[1] = None
    tight = experts()
    tight.part_stride[2] -= 2
    yield from (none, two, part, tight, experts(n_experts=0), experts(n_experts=513), experts(d_model=0), experts(w_type=ops.F32),
                experts(d_ff=1 << 24), experts(w_type=ops.Q4, d_model=48))
    shape = view()
    shape.parts[1].bytes -= 2
    base = view()
    base.parts[0].base = None
    for v in (view(n_parts=2), view(n_gated=1), view(slot_of=None), view(struct_size=16), shape, base):
        e = experts(view=C.pointer(v), gated=1)
        e.part[0] = None
        yield e


@pytest.mark.parametrize("i", range(16))
def test_experts(i):
    e = list(bad_experts())[i]
    a = ops.TsaFfnArgs(x=P, x_stride=64, ids=P, weights=P, y=P, y_stride=64, rows=2, top_k=2, type=ops.BF16, act=1)
    refused(ops._ops().tsa_ffn, C.byref(e), C.byref(a), P, 1 << 40, None, says="tsa_ffn")


def test_ffn():
    f, e = ops._ops().tsa_ffn, experts()
    a = ops.TsaFfnArgs(x=P, x_stride=64, ids=P, weights=P, y=P, y_stride=64, rows=2, top_k=2, type=ops.BF16, act=1)
    refused(f, None, C.byref(a), P, 1 << 40, None)
    refused(f, C.byref(e), None, P, 1 << 40, None)
    for bad in (dict(type=ops.F32), dict(type=ops.F16), dict(act=0), dict(act=9), dict(top_k=0), dict(top_k=65), dict(ids=None),
                dict(ids=P + 2), dict(weights=P + 1), dict(rows=1 << 23), dict(x=None), dict(x_stride=63), dict(y=None), dict(y=P + 1),
                dict(residual=P, residual_stride=1)):
        refused(f, C.byref(e), C.byref(changed(a, **bad)), P, 1 << 40, None, says="tsa_ffn")
    need = ops._ops().tsa_ffn_workspace(C.byref(e), 2, 2)
    assert need > 0
    refused(f, C.byref(e), C.byref(a), P, need - 1, None, says="workspace")
    refused(f, C.byref(e), C.byref(a), None, need, None, says="workspace")
    assert ops._ops().tsa_ffn_workspace(C.byref(e), 2, 0) == 0
    assert f(C.byref(e), C.byref(changed(a, rows=0, x=None)), None, 0, None) == tsa.SS_OK


def test_ffn_backward():
    f, e = ops._ops().tsa_ffn_backward, experts()
    a = ops.TsaFfnGradArgs(x=P, x_stride=64, ids=P, weights=P, dy=P, dy_stride=64, dx=P, dx_stride=64, rows=2, top_k=2,
                           type=ops.BF16, act=1)
    refused(f, C.byref(experts(w_type=ops.Q4)), C.byref(a), P, 1 << 40, None, status=tsa.SS_E_UNSUPPORTED, says="4-bit")
    for bad in (dict(dgate=P), dict(dgate=P, dup=P), dict(dgate=P, dup=P, ddown=P + 1), dict(dy=None), dict(dy_stride=9), dict(dx=P + 1),
                dict(dweights=P + 2), dict(type=ops.F16), dict(act=0)):
        refused(f, C.byref(e), C.byref(changed(a, **bad)), P, 1 << 40, None, says="tsa_ffn_backward")
    need = ops._ops().tsa_ffn_backward_workspace(C.byref(e), 2, 2)
    refused(f, C.byref(e), C.byref(a), P, need - 1, None, says="workspace")


class Fake:
    """An array object without memory: what ops looks at."""

    def __init__(self, *shape, dtype="torch.bfloat16", stride=None):
        self.shape, self.dtype, self.s = shape, dtype, stride or (shape[-1], 1)

    def stride(self):
        return self.s

    def data_ptr(self):
        return P

    def is_contiguous(self):
        return self.s == (self.shape[-1], 1)

    def numel(self):
        return 1 << 20

    def element_size(self):
        return 2


def test_python_side():
    x, w, y = Fake(2, 128), Fake(64, 128), Fake(2, 64)
    for bad in (lambda: ops.linear(x, Fake(64, 120), y), lambda: ops.linear(x, w, Fake(3, 64)), lambda: ops.linear(Fake(2, 128, stride=(1, 2)), w, y),
                lambda: ops.linear(x, w, y, bias=Fake(64, dtype="torch.float32", stride=(1,))), lambda: ops.linear(x, w, y, residual=Fake(2, 64, dtype="torch.float32")),
                lambda: ops.linear(Fake(2, 120), Fake(64, 72, dtype="torch.uint8"), y),
                lambda: ops.route(Fake(2, 64, dtype="torch.float32"), Fake(3, 8, dtype="torch.int32"), Fake(2, 8, dtype="torch.float32"))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(KeyError):
        ops.linear(x, w, y, act="swish")
    with pytest.raises(tsa.SsError) as e:
        ops.linear(x, Fake(64, 128, dtype="torch.float16"), y)
    assert e.value.status == tsa.SS_E_INVALID
