"""The model operators of include/tierstream_amd/tsa_ops.h, on any 2-D array objects that have data_ptr(), shape, stride()
and dtype as torch's tensors have (torch itself is not imported), all in device memory: what says by is_cuda that it is
elsewhere is refused. Streams are hipStream_t handles (torch.cuda.current_stream().cuda_stream); outputs and workspaces are
the caller's. Errors are raised as SsError, arrays that do not fit together or are not the device's as ValueError.

    ops.route(logits, ids, weights, stream=s)                       # ids for ss_dg_enqueue_export and for ops.ffn
    e = ops.Experts.in_arena(ctx.dg_view(), g, n, d, f, "bf16")     # the slots of gated layer g
    ops.ffn(e, x, y, ids=ids, weights=weights, residual=x0, workspace=ws, stream=s)
"""
from __future__ import annotations

import ctypes as C

from . import check, lib
from .ss import SsDgDeviceView

vp, u32, u64 = C.c_void_p, C.c_uint32, C.c_uint64

BF16, F16, F32, Q4 = range(4)
ACTS = {"none": 0, "silu": 1, "gelu": 2, "gelu_tanh": 3, "relu": 4}
_TYPES = {"bf16": BF16, "f16": F16, "f32": F32, "q4": Q4, "torch.bfloat16": BF16, "torch.float16": F16,
          "torch.float32": F32, "torch.uint8": Q4}
_Q4_BLOCK, _Q4_BYTES = 32, 18


class TsaRouteArgs(C.Structure):
    _fields_ = [("logits", vp), ("logits_stride", u64), ("ids", vp), ("weights", vp), ("rows", u32), ("n_experts", u32),
                ("top_k", u32), ("type", u32), ("renorm", u32), ("scale", C.c_float)]


class TsaLinearArgs(C.Structure):
    _fields_ = [("x", vp), ("x_stride", u64), ("w", vp), ("w_stride", u64), ("bias", vp), ("residual", vp),
                ("residual_stride", u64), ("y", vp), ("y_stride", u64), ("rows", u32), ("n_in", u32), ("n_out", u32),
                ("x_type", u32), ("w_type", u32), ("y_type", u32), ("act", u32), ("reserved", u32)]


class TsaExperts(C.Structure):
    _fields_ = [("n_experts", u32), ("d_model", u32), ("d_ff", u32), ("w_type", u32), ("part", vp * 3),
                ("part_stride", u64 * 3), ("table", vp), ("view", C.POINTER(SsDgDeviceView)), ("gated", u32),
                ("reserved", u32)]


class TsaFfnArgs(C.Structure):
    _fields_ = [("x", vp), ("x_stride", u64), ("ids", vp), ("weights", vp), ("residual", vp), ("residual_stride", u64),
                ("y", vp), ("y_stride", u64), ("rows", u32), ("top_k", u32), ("type", u32), ("act", u32)]


class TsaFfnGradArgs(C.Structure):
    _fields_ = [("x", vp), ("x_stride", u64), ("ids", vp), ("weights", vp), ("dy", vp), ("dy_stride", u64), ("dx", vp),
                ("dx_stride", u64), ("dweights", vp), ("dgate", vp), ("dup", vp), ("ddown", vp), ("rows", u32),
                ("top_k", u32), ("type", u32), ("act", u32)]


_lib = None


def _ops() -> C.CDLL:
    global _lib
    if _lib is None:
        L, st = lib(), C.c_int
        sigs = {
            "tsa_route": (st, [C.POINTER(TsaRouteArgs), vp]),
            "tsa_route_backward": (st, [C.POINTER(TsaRouteArgs), vp, vp, u64, vp]),
            "tsa_linear_workspace": (u64, [C.POINTER(TsaLinearArgs)]),
            "tsa_linear": (st, [C.POINTER(TsaLinearArgs), vp, u64, vp]),
            "tsa_ffn_workspace": (u64, [C.POINTER(TsaExperts), u32, u32]),
            "tsa_ffn": (st, [C.POINTER(TsaExperts), C.POINTER(TsaFfnArgs), vp, u64, vp]),
            "tsa_ffn_backward_workspace": (u64, [C.POINTER(TsaExperts), u32, u32]),
            "tsa_ffn_backward": (st, [C.POINTER(TsaExperts), C.POINTER(TsaFfnGradArgs), vp, u64, vp]),
        }
        for name, (res, args) in sigs.items():
            f = getattr(L, name)
            f.restype, f.argtypes = res, args
        _lib = L
    return _lib


# Calls of a decode step take microseconds on the device: what runs on the host for each is kept short. Names of types are
# looked up once per type.
_of_dtype: dict = {}


def _type(t) -> int:
    d = t.dtype
    kind = _of_dtype.get(d)
    if kind is None:
        kind = _of_dtype[d] = _TYPES[str(d)]
    return kind


def _device(t, what: str) -> None:
    """A kernel takes an address as it is: one of the host's would fault the device."""
    if not getattr(t, "is_cuda", True):
        raise ValueError(f"{what}: not in device memory")


def _mat(t, rows: int, cols: int, what: str, kind: int | None = None):
    """(pointer, row stride) of a matrix with contiguous rows."""
    stride = t.stride()
    if t.shape != (rows, cols) or (cols > 1 and stride[1] != 1):
        raise ValueError(f"{what}: a [{rows}][{cols}] matrix with contiguous rows, not {tuple(t.shape)}")
    _device(t, what)
    if kind is not None and _type(t) != kind:
        raise ValueError(f"{what}: another type than the operator's ({t.dtype})")
    return t.data_ptr(), stride[0]


_dtype_named: dict = {}


def _vec(t, shape, dtype: str, what: str):
    """Pointer of a contiguous array."""
    if t is None:
        return None
    d = t.dtype
    name = _dtype_named.get(d)
    if name is None:
        name = _dtype_named[d] = str(d)
    if t.shape != shape or name != dtype or not t.is_contiguous():
        raise ValueError(f"{what}: a contiguous {dtype} array of {tuple(shape)}, not {t.dtype} {tuple(t.shape)}")
    _device(t, what)
    return t.data_ptr()


def _ok(status: int) -> None:
    if status:
        check(status)


def _room(workspace):
    if workspace is None:
        return None, 0
    _device(workspace, "workspace")
    return workspace.data_ptr(), workspace.numel() * workspace.element_size()


# ---- the choice of experts -------------------------------------------------------------------------------------------
def _route_args(logits, ids, weights, renorm, scale):
    rows, n = logits.shape
    shape = (rows, ids.shape[1])
    p, stride = _mat(logits, rows, n, "logits")
    return TsaRouteArgs(p, stride, _vec(ids, shape, "torch.int32", "ids"), _vec(weights, shape, "torch.float32", "weights"), rows, n,
                        shape[1], _type(logits), renorm, scale)


def route(logits, ids, weights, *, renorm=True, scale=1.0, stream=None) -> None:
    """ids int32 [rows][top_k] and weights float32 [rows][top_k] of each row's largest logits (tsa_route)."""
    _ok(_ops().tsa_route(_route_args(logits, ids, weights, renorm, scale), stream))


def route_backward(logits, ids, dweights, dlogits, *, renorm=True, scale=1.0, stream=None) -> None:
    """dlogits (the logits' type) from dweights (tsa_route_backward)."""
    a = _route_args(logits, ids, None, renorm, scale)
    p, stride = _mat(dlogits, a.rows, a.n_experts, "dlogits", a.type)
    _ok(_ops().tsa_route_backward(a, _vec(dweights, ids.shape, "torch.float32", "dweights"), p, stride, stream))


# ---- products ----------------------------------------------------------------------------------------------------------
def _linear_args(x, w, y, bias=None, residual=None, act="none"):
    (rows, n_in), n_out = x.shape, w.shape[0]
    kind, w_kind, y_kind = _type(x), _type(w), _type(y)
    xp, xs = _mat(x, rows, n_in, "x")
    if w_kind == Q4:
        if n_in % _Q4_BLOCK or not w.is_contiguous():
            raise ValueError("w: 4-bit weights are whole blocks of 32 values, rows back to back")
        wp, ws = _mat(w, n_out, n_in // _Q4_BLOCK * _Q4_BYTES, "w")[0], n_in
    else:
        wp, ws = _mat(w, n_out, n_in, "w")
    yp, ys = _mat(y, rows, n_out, "y")
    rp, rs = (None, 0) if residual is None else _mat(residual, rows, n_out, "residual", y_kind)
    bp = None if bias is None else _vec(bias, (n_out,), str(x.dtype), "bias")
    return TsaLinearArgs(xp, xs, wp, ws, bp, rp, rs, yp, ys, rows, n_in, n_out, kind, w_kind, y_kind, ACTS[act], 0)


def linear_workspace(x, w, y) -> int:
    """Workspace bytes of linear(x, w, y, ...)."""
    rows, n_in = x.shape
    kind = _type(w)
    a = TsaLinearArgs(x.data_ptr(), x.stride()[0], w.data_ptr(), n_in if kind == Q4 else w.stride()[0], None, None, 0, None, 0, rows,
                      n_in, w.shape[0], _type(x), kind, _type(y), 0, 0)
    return _ops().tsa_linear_workspace(a)


def linear(x, w, y, *, bias=None, residual=None, act="none", workspace=None, stream=None) -> None:
    """y = act(x w^T + bias) + residual (tsa_linear). w: [n_out][n_in] of x's type, or uint8 [n_out][n_in / 32 * 18]."""
    a = _linear_args(x, w, y, bias, residual, act)
    ws, n = _room(workspace)
    _ok(_ops().tsa_linear(a, ws, n, stream))


# ---- gated feed-forward blocks --------------------------------------------------------------------------------------------
class Experts:
    """Where a layer's gate, up and down weights are (tsa_experts)."""

    def __init__(self, n_experts: int, d_model: int, d_ff: int, kind: str | int):
        self.s = TsaExperts(n_experts=n_experts, d_model=d_model, d_ff=d_ff,
                            w_type=_TYPES[kind] if isinstance(kind, str) else kind)
        self.keep = None  # what the struct points to

    @classmethod
    def stacked(cls, gate, up, down) -> "Experts":
        """gate, up [n][d_ff][d_model], down [n][d_model][d_ff] (uint8: rows of 4-bit blocks), each contiguous."""
        n, f, width = gate.shape
        kind = _type(gate)
        if kind == Q4 and (width % _Q4_BYTES or f % _Q4_BLOCK):
            raise ValueError(f"gate: 4-bit rows are whole blocks of {_Q4_BYTES} bytes and d_ff a multiple of {_Q4_BLOCK}, not {f} rows of {width} bytes")
        d = width // _Q4_BYTES * _Q4_BLOCK if kind == Q4 else width
        wide = f // _Q4_BLOCK * _Q4_BYTES if kind == Q4 else f
        for t, shape, what in ((gate, (n, f, width), "gate"), (up, (n, f, width), "up"), (down, (n, d, wide), "down")):
            if tuple(t.shape) != shape or t.dtype != gate.dtype or not t.is_contiguous():
                raise ValueError(f"{what}: a contiguous array of {shape}, not {tuple(t.shape)} {t.dtype}")
            _device(t, what)
        e = cls(n, d, f, kind)
        e.keep = (gate, up, down)
        for p, t in enumerate(e.keep):
            e.s.part[p], e.s.part_stride[p] = t.data_ptr(), t.stride(0) * t.element_size()
        return e

    @classmethod
    def in_table(cls, table, d_model: int, d_ff: int, kind: str) -> "Experts":
        """table: int64 / uint64 [n] of unit addresses on the device (ss_layer_view.table_dev), each 0 or 16-byte aligned."""
        if len(table.shape) != 1 or str(table.dtype) not in ("torch.int64", "torch.uint64") or not table.is_contiguous():
            raise ValueError(f"table: a contiguous array of 64-bit addresses, not {table.dtype} {tuple(table.shape)}")
        _device(table, "table")
        e = cls(table.numel(), d_model, d_ff, kind)
        e.keep = table
        e.s.table = table.data_ptr()
        return e

    @classmethod
    def in_arena(cls, view: SsDgDeviceView, gated: int, n_experts: int, d_model: int, d_ff: int, kind: str) -> "Experts":
        """The slots of a device-gated context's gated layer (Ctx.dg_view())."""
        e = cls(n_experts, d_model, d_ff, kind)
        e.keep = view
        e.s.view, e.s.gated = C.pointer(view), gated
        return e


def ffn_workspace(e: Experts, rows: int, top_k: int = 1) -> int:
    return _ops().tsa_ffn_workspace(e.s, rows, top_k)


def _pairs(a, e: Experts, x, ids, weights):
    rows, d = x.shape
    if d != e.s.d_model:
        raise ValueError(f"x: rows of d_model = {e.s.d_model} values, not {d}")
    a.x, a.x_stride = _mat(x, rows, d, "x")
    a.rows, a.top_k, a.type = rows, 1 if ids is None else ids.shape[1], _type(x)
    shape = (rows, a.top_k)
    a.ids, a.weights = _vec(ids, shape, "torch.int32", "ids"), _vec(weights, shape, "torch.float32", "weights")
    return rows, d


def ffn(e: Experts, x, y, *, ids=None, weights=None, residual=None, act="silu", workspace=None, stream=None) -> None:
    """y_t = residual_t + sum_j weights_tj expert_{ids_tj}(x_t) (tsa_ffn); ids None: every row through expert 0."""
    a = TsaFfnArgs(act=ACTS[act])
    rows, d = _pairs(a, e, x, ids, weights)
    a.y, a.y_stride = _mat(y, rows, d, "y", a.type)
    if residual is not None:
        a.residual, a.residual_stride = _mat(residual, rows, d, "residual", a.type)
    ws, n = _room(workspace)
    _ok(_ops().tsa_ffn(e.s, a, ws, n, stream))


def ffn_backward_workspace(e: Experts, rows: int, top_k: int = 1) -> int:
    return _ops().tsa_ffn_backward_workspace(e.s, rows, top_k)


def ffn_backward(e: Experts, x, dy, dx=None, *, ids=None, weights=None, dweights=None, dgate=None, dup=None, ddown=None,
                 act="silu", workspace=None, stream=None) -> None:
    """The gradients of ffn for dy that are asked for (tsa_ffn_backward)."""
    a = TsaFfnGradArgs(act=ACTS[act])
    rows, d = _pairs(a, e, x, ids, weights)
    a.dy, a.dy_stride = _mat(dy, rows, d, "dy", a.type)
    if dx is not None:
        a.dx, a.dx_stride = _mat(dx, rows, d, "dx", a.type)
    a.dweights = _vec(dweights, (rows, a.top_k), "torch.float32", "dweights")
    n, f = e.s.n_experts, e.s.d_ff
    a.dgate = _vec(dgate, (n, f, d), str(x.dtype), "dgate")
    a.dup = _vec(dup, (n, f, d), str(x.dtype), "dup")
    a.ddown = _vec(ddown, (n, d, f), str(x.dtype), "ddown")
    ws, n = _room(workspace)
    _ok(_ops().tsa_ffn_backward(e.s, a, ws, n, stream))
