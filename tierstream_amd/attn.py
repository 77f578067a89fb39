"""The attention operators of include/tierstream_amd/tsa_attn.h, on array objects as tierstream_amd.ops takes them (data_ptr(), shape,
stride(), dtype and device as torch's tensors have), all in the memory of the current device, to which the stream belongs too. Queries, keys and values are [tokens][heads][head_dim] with contiguous
values and any strides of tokens and heads, so that slices of one product's output go as they are. Streams are hipStream_t
handles; outputs and workspaces are the caller's. Errors are raised as SsError, arrays that do not fit together as ValueError.

    rotary = attn.Rotary(128, base=1e6)
    cache = attn.Cache(pages, kv_heads, 128)                        # uint8 [n_pages][kv_heads][attn.page_bytes(128)]
    attn.plan(lengths, fresh, table, free, n_free, first, positions, slots, status, stream=s)  # lengths, n_free: as they are then
    attn.rotate(rotary, positions, q, k, stream=s)                  # in place
    attn.store(cache, k, v, slots, stream=s)
    attn.attend_cached(cache, q, out, table, lengths, first, workspace=ws, stream=s)
"""
from __future__ import annotations

import ctypes as C
import struct

from . import lib
from .ops import _device, _ok, _room, _type, _vec

vp, u32, u64, f64 = C.c_void_p, C.c_uint32, C.c_uint64, C.c_double

PAGE = 64  # tokens of a page
MAX_PAIRS = 128


class TsaHeads(C.Structure):
    _fields_ = [("p", vp), ("token_stride", u64), ("head_stride", u64), ("heads", u32), ("reserved", u32)]


class TsaRotaryParams(C.Structure):
    _fields_ = [("base", f64), ("factor", f64), ("trained", f64), ("low", f64), ("high", f64), ("amplitude", f64), ("rotated", u32),
                ("interleaved", u32)]


class TsaRotary(C.Structure):
    _fields_ = [("turns", f64 * MAX_PAIRS), ("amplitude", f64), ("pairs", u32), ("interleaved", u32)]


class TsaRotateArgs(C.Structure):
    _fields_ = [("x", TsaHeads * 2), ("y", TsaHeads * 2), ("positions", vp), ("tokens", u32), ("head_dim", u32), ("type", u32),
                ("backward", u32)]


class TsaCache(C.Structure):
    _fields_ = [("pages", vp), ("n_pages", u32), ("kv_heads", u32), ("head_dim", u32), ("reserved", u32)]


class TsaCachePlanArgs(C.Structure):
    _fields_ = [("lengths", vp), ("fresh", vp), ("table", vp), ("table_stride", u64), ("free", vp), ("n_free", vp), ("ends", vp), ("left", vp),
                ("first", vp), ("positions", vp), ("slots", vp), ("status", vp), ("requests", u32), ("width", u32), ("pages", u32),
                ("rows", u32)]


class TsaCacheRowsArgs(C.Structure):
    _fields_ = [("k", TsaHeads), ("v", TsaHeads), ("slots", vp), ("tokens", u32), ("type", u32)]


class TsaAttendCachedArgs(C.Structure):
    _fields_ = [("q", TsaHeads), ("out", TsaHeads), ("table", vp), ("table_stride", u64), ("ends", vp), ("first", vp), ("tokens", u32),
                ("requests", u32), ("width", u32), ("type", u32), ("scale", C.c_float), ("reserved", u32)]


class TsaAttendArgs(C.Structure):
    _fields_ = [("q", TsaHeads), ("k", TsaHeads), ("v", TsaHeads), ("out", TsaHeads), ("first", vp), ("k_first", vp), ("lse", vp),
                ("tokens", u32), ("k_tokens", u32), ("sequences", u32), ("head_dim", u32), ("type", u32), ("causal", u32),
                ("scale", C.c_float), ("reserved", u32)]


class TsaAttendGradArgs(C.Structure):
    _fields_ = [("f", TsaAttendArgs), ("dout", TsaHeads), ("dq", TsaHeads), ("dk", TsaHeads), ("dv", TsaHeads)]


_lib = None


def _attn() -> C.CDLL:
    global _lib
    if _lib is None:
        L, st, P = lib(), C.c_int, C.POINTER
        sigs = {
            "tsa_rotary_init": (st, [P(TsaRotaryParams), P(TsaRotary)]),
            "tsa_rotate": (st, [P(TsaRotary), P(TsaRotateArgs), vp]),
            "tsa_cache_plan": (st, [P(TsaCachePlanArgs), vp]),
            "tsa_cache_slots": (st, [P(TsaCachePlanArgs), vp]),
            "tsa_cache_store": (st, [P(TsaCache), P(TsaCacheRowsArgs), vp]),
            "tsa_cache_load": (st, [P(TsaCache), P(TsaCacheRowsArgs), vp]),
            "tsa_attend_cached_workspace": (u64, [P(TsaCache), P(TsaAttendCachedArgs)]),
            "tsa_attend_cached": (st, [P(TsaCache), P(TsaAttendCachedArgs), vp, u64, vp]),
            "tsa_attend": (st, [P(TsaAttendArgs), vp]),
            "tsa_attend_backward_workspace": (u64, [P(TsaAttendArgs)]),
            "tsa_attend_backward": (st, [P(TsaAttendGradArgs), vp, u64, vp]),
        }
        for name, (res, args) in sigs.items():
            f = getattr(L, name)
            f.restype, f.argtypes = res, args
        _lib = L
    return _lib


# A decode step's calls take microseconds on the device: what runs on the host for each is kept short. Structs are packed as
# bytes (one of four tsa_heads: 1 us, field by field 6), and the calls that take them are functions of their own.
_ROTATE, _PLAN = struct.Struct("QQQII" * 4 + "QIIII"), struct.Struct("QQQQQQQQQQQQIIII")
_ROWS, _CACHED = struct.Struct("QQQII" * 2 + "QII"), struct.Struct("QQQII" * 2 + "QQQQIIIIfI")
_ATTEND, _GRAD = struct.Struct("QQQII" * 4 + "QQQIIIIIIfI"), struct.Struct("QQQII" * 4 + "QQQIIIIIIfI" + "QQQII" * 4)
_NONE = (0, 0, 0, 0, 0)
_calls: dict = {}


def _call(name: str):
    f = _calls.get(name)
    if f is None:
        declared, f = getattr(_attn(), name), _attn()[name]
        f.restype, f.argtypes = declared.restype, [C.c_char_p if issubclass(t, C._Pointer) else t for t in declared.argtypes]
        _calls[name] = f
    return f


def _apart(what: str, *devices) -> None:
    for d in devices[1:]:
        if d != devices[0]:
            raise ValueError(f"{what}: arrays on {devices[0]} and on {d}")


def _heads(t, what: str, shape=None, dtype=None) -> tuple:
    """A tsa_heads of [tokens][heads][head_dim] with contiguous values."""
    n = t.shape
    if shape is not None and n != shape:
        raise ValueError(f"{what}: [tokens][heads][head_dim] of {tuple(shape)}, not {tuple(n)}")
    if len(n) != 3:
        raise ValueError(f"{what}: [tokens][heads][head_dim], not {tuple(n)}")
    by_token, by_head, by_value = t.stride()
    if by_value != 1 and n[2] > 1:
        raise ValueError(f"{what}: the values of a head lie next to each other")
    if not getattr(t, "is_cuda", True):
        raise ValueError(f"{what}: not in device memory")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{what}: another type than the operator's ({t.dtype})")
    return t.data_ptr(), by_token, by_head, n[1], 0


_int32: dict = {}


def _ints(t, n: int, what: str) -> int:
    """Pointer of n contiguous 32-bit integers."""
    is_int32 = _int32.get(t.dtype)
    if is_int32 is None:
        is_int32 = _int32[t.dtype] = str(t.dtype) == "torch.int32"
    if t.shape != (n,) or not is_int32 or not t.is_contiguous():
        raise ValueError(f"{what}: {n} contiguous 32-bit integers, not {t.dtype} {tuple(t.shape)}")
    if not getattr(t, "is_cuda", True):
        raise ValueError(f"{what}: not in device memory")
    return t.data_ptr()


def _three(t, what: str):
    n = t.shape
    if len(n) != 3:
        raise ValueError(f"{what}: [tokens][heads][head_dim], not {tuple(n)}")
    return n


# ---- rotary positions ----------------------------------------------------------------------------------------------------
class Rotary:
    """How positions turn the first `rotated` values of a head (tsa_rotary_params)."""

    def __init__(self, rotated: int, *, base=10000.0, interleaved=False, factor=1.0, trained=0, low=1.0, high=4.0, amplitude=1.0):
        self.s = TsaRotary()
        _ok(_attn().tsa_rotary_init(TsaRotaryParams(base, factor, trained, low, high, amplitude, rotated, interleaved), self.s))
        self.packed = bytes(self.s)


def rotate(rotary: Rotary, positions, q, k=None, q_out=None, k_out=None, *, backward=False, stream=None) -> None:
    """q, and k if there is one, turned by positions int32 [tokens] (tsa_rotate): in place, or to q_out and k_out. backward: the gradients of
    what was turned become those of what it was made from."""
    x, dtype, device = _heads(q, "q"), q.dtype, q.device
    tokens, heads, dim = q.shape
    y, u, v = x, _NONE, _NONE
    at = _ints(positions, tokens, "positions")
    _apart("rotate", device, positions.device)
    if q_out is not None:
        y = _heads(q_out, "q_out", q.shape, dtype)
        _apart("rotate", device, q_out.device)
    if k is not None:
        u = v = _heads(k, "k", (tokens, _three(k, "k")[1], dim), dtype)
        _apart("rotate", device, k.device)
        if k_out is not None:
            v = _heads(k_out, "k_out", k.shape, dtype)
            _apart("rotate", device, k_out.device)
    elif k_out is not None:
        raise ValueError("k_out without k")
    _ok(_call("tsa_rotate")(rotary.packed, _ROTATE.pack(*x, *u, *y, *v, at, tokens, dim, _type(q), backward), stream))


# ---- the cache -----------------------------------------------------------------------------------------------------------
def page_bytes(head_dim: int) -> int:
    """Bytes of a page of one head."""
    return 72 * head_dim


class Cache:
    """Pages of 4-bit keys and values: uint8 [n_pages][kv_heads][page_bytes(head_dim)], contiguous. Nothing has to be cleared."""

    def __init__(self, pages, kv_heads: int, head_dim: int):
        n = pages.shape[0]
        p = _vec(pages, (n, kv_heads, page_bytes(head_dim)), "torch.uint8", "pages")
        self.pages, self.device, self.s = pages, pages.device, TsaCache(p, n, kv_heads, head_dim)
        self.kv_heads, self.head_dim, self.packed = kv_heads, head_dim, bytes(self.s)


def _table(table, n: int):
    shape = table.shape
    if len(shape) != 2 or not _int32.get(table.dtype, str(table.dtype) == "torch.int32") or (shape[1] > 1 and table.stride()[1] != 1):
        raise ValueError(f"table: int32 [requests][pages] with contiguous rows, not {table.dtype} {tuple(shape)}")
    if shape[0] != n:
        raise ValueError(f"table: a row for each of {n} requests, not {shape[0]}")
    _device(table, "table")
    return table.data_ptr(), table.stride()[0], shape[1]


def plan(lengths, fresh, table, free, n_free, first, positions, slots, status, *, ends=None, left=None, stream=None) -> None:
    """Pages, positions and slots of a step (tsa_cache_plan), all int32: lengths, fresh [requests], table [requests][pages], free [pages],
    n_free [1], first [requests + 1], positions and slots [rows], status [1]. ends and left None: lengths and n_free become them."""
    ends, left = lengths if ends is None else ends, n_free if left is None else left
    n, rows, pages = lengths.shape[0], positions.shape[0], free.shape[0]
    t, stride, width = _table(table, n)
    packed = _PLAN.pack(_ints(lengths, n, "lengths"), _ints(fresh, n, "fresh"), t, stride, _ints(free, pages, "free"), _ints(n_free, 1, "n_free"),
                        _ints(ends, n, "ends"), _ints(left, 1, "left"), _ints(first, n + 1, "first"), _ints(positions, rows, "positions"),
                        _ints(slots, rows, "slots"), _ints(status, 1, "status"), n, width, pages, rows)
    _apart("plan", lengths.device, fresh.device, table.device, free.device, n_free.device, ends.device, left.device, first.device, positions.device,
           slots.device, status.device)
    _ok(_call("tsa_cache_plan")(packed, stream))


def slots(table, ends, first, positions, out, *, stream=None) -> None:
    """Positions and slots (out) of the rows first[i]..first[i + 1], the last tokens of request i's ends[i] (tsa_cache_slots)."""
    n, rows = ends.shape[0], positions.shape[0]
    t, stride, width = _table(table, n)
    packed = _PLAN.pack(0, 0, t, stride, 0, 0, _ints(ends, n, "ends"), 0, _ints(first, n + 1, "first"), _ints(positions, rows, "positions"),
                        _ints(out, rows, "slots"), 0, n, width, 0, rows)
    _apart("slots", table.device, ends.device, first.device, positions.device, out.device)
    _ok(_call("tsa_cache_slots")(packed, stream))


def _rows(cache: Cache, k, v, slots, what: str) -> bytes:
    tokens = _three(k, "k")[0]
    shape = (tokens, cache.kv_heads, cache.head_dim)
    packed = _ROWS.pack(*_heads(k, "k", shape), *_heads(v, "v", shape, k.dtype), _ints(slots, tokens, "slots"), tokens, _type(k))
    _apart(what, cache.device, k.device, v.device, slots.device)
    return packed


def store(cache: Cache, k, v, slots, *, stream=None) -> None:
    """Keys and values [tokens][kv_heads][head_dim] to slots int32 [tokens] as 4-bit values (tsa_cache_store)."""
    _ok(_call("tsa_cache_store")(cache.packed, _rows(cache, k, v, slots, "store"), stream))


def load(cache: Cache, slots, k, v, *, stream=None) -> None:
    """What the slots hold to k and v (tsa_cache_load)."""
    _ok(_call("tsa_cache_load")(cache.packed, _rows(cache, k, v, slots, "load"), stream))


def attend_cached_workspace(cache: Cache, q, table) -> int:
    """Workspace bytes of attend_cached; grows with q's rows and the table's requests and width."""
    (tokens, heads, _), (n, width) = q.shape, table.shape
    return _call("tsa_attend_cached_workspace")(cache.packed, _CACHED.pack(0, 0, 0, heads, 0, *_NONE, 0, 0, 0, 0, tokens, n, width, _type(q), 0.0, 0))


def attend_cached(cache: Cache, q, out, table, ends, first, *, scale=None, workspace=None, stream=None) -> None:
    """out = softmax(q K^T scale) V over the pages of each row's request (tsa_attend_cached). scale None: head_dim^-0.5."""
    x, n = _heads(q, "q"), ends.shape[0]
    tokens, _, dim = q.shape
    if dim != cache.head_dim:
        raise ValueError(f"q: heads of the cache's {cache.head_dim} values, not {dim}")
    t, stride, width = _table(table, n)
    packed = _CACHED.pack(*x, *_heads(out, "out", q.shape, q.dtype), t, stride, _ints(ends, n, "ends"), _ints(first, n + 1, "first"), tokens, n, width,
                          _type(q), dim ** -0.5 if scale is None else scale, 0)
    ws, size = _room(workspace)
    _apart("attend_cached", cache.device, q.device, out.device, table.device, ends.device, first.device, cache.device if ws is None else workspace.device)
    _ok(_call("tsa_attend_cached")(cache.packed, packed, ws, size, stream))


# ---- packed sequences ----------------------------------------------------------------------------------------------------
def _attend_fields(what, q, k, v, out, lse, first, k_first, causal, scale) -> tuple:
    x, dtype, device = _heads(q, "q"), q.dtype, q.device
    (tokens, heads, dim), (k_tokens, kept, _) = q.shape, _three(k, "k")
    shape, n = (k_tokens, kept, dim), 1 if first is None else first.shape[0] - 1
    if n < 0:
        raise ValueError("first: [sequences + 1], not []")
    fields = (*x, *_heads(k, "k", shape, dtype), *_heads(v, "v", shape, dtype), *_heads(out, "out", q.shape, dtype),
              0 if first is None else _ints(first, n + 1, "first"), 0 if k_first is None else _ints(k_first, n + 1, "k_first"),
              0 if lse is None else _vec(lse, (heads, tokens), "torch.float32", "lse"), tokens, k_tokens, n, dim, _type(q), causal,
              dim ** -0.5 if scale is None else scale, 0)
    _apart(what, device, k.device, v.device, out.device, *[t.device for t in (lse, first, k_first) if t is not None])
    return fields


def attend(q, k, v, out, *, lse=None, first=None, k_first=None, causal=True, scale=None, stream=None) -> None:
    """out = softmax(q K^T scale) V over packed sequences (tsa_attend); lse: float32 [heads][tokens]; first, k_first: int32
    [sequences + 1] (None: one sequence). scale None: head_dim^-0.5."""
    _ok(_call("tsa_attend")(_ATTEND.pack(*_attend_fields("attend", q, k, v, out, lse, first, k_first, causal, scale)), stream))


def attend_backward_workspace(q, k) -> int:
    """Workspace bytes of attend_backward; grows with the rows."""
    (tokens, heads, dim), (k_tokens, kept, _) = q.shape, k.shape
    return _call("tsa_attend_backward_workspace")(_ATTEND.pack(0, 0, 0, heads, 0, 0, 0, 0, kept, 0, 0, 0, 0, kept, 0, *_NONE, 0, 0, 0, tokens, k_tokens, 1,
                                                               dim, _type(q), 0, 0.0, 0))


def attend_backward(q, k, v, out, dout, lse, dq=None, dk=None, dv=None, *, first=None, k_first=None, causal=True, scale=None,
                    workspace=None, stream=None) -> None:
    """The gradients of attend for dout that are asked for (tsa_attend_backward), from its inputs, out and lse."""
    fields, dtype = _attend_fields("attend_backward", q, k, v, out, lse, first, k_first, causal, scale), q.dtype
    grads = [_NONE if t is None else _heads(t, name, like.shape, dtype) for t, name, like in ((dq, "dq", q), (dk, "dk", k), (dv, "dv", v))]
    packed = _GRAD.pack(*fields, *_heads(dout, "dout", q.shape, dtype), *grads[0], *grads[1], *grads[2])
    ws, size = _room(workspace)
    _apart("attend_backward", q.device, dout.device, *[t.device for t in (dq, dk, dv, workspace) if t is not None])
    _ok(_call("tsa_attend_backward")(packed, ws, size, stream))
