"""The attention operators of include/tierstream_amd/tsa_attn.h, on array objects as tierstream_amd.ops takes them (data_ptr(), shape,
stride() and dtype as torch's tensors have), all in device memory and on the same device. Queries, keys and values are [tokens][heads][head_dim] with contiguous
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

from . import lib
from .ops import F32, _device, _ok, _room, _type, _vec

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


def _same_device(what: str, *arrays) -> None:
    """One device holds all that a call reads and writes."""
    at = None
    for t in arrays:
        d = getattr(t, "device", None)
        if d is not None:
            if at is not None and d != at:
                raise ValueError(f"{what}: arrays on {at} and on {d}")
            at = d


def _three(t, what: str):
    n = t.shape
    if len(n) != 3:
        raise ValueError(f"{what}: [tokens][heads][head_dim], not {tuple(n)}")
    return n


def _heads(t, what: str, shape=None, kind: int | None = None) -> tuple:
    """(pointer, token stride, head stride, heads) of [tokens][heads][head_dim] with contiguous values."""
    n = _three(t, what)
    if shape is not None and tuple(n) != tuple(shape):
        raise ValueError(f"{what}: [tokens][heads][head_dim] of {tuple(shape)}, not {tuple(n)}")
    stride = t.stride()
    if n[2] > 1 and stride[2] != 1:
        raise ValueError(f"{what}: the values of a head lie next to each other")
    _device(t, what)
    if kind is not None and _type(t) != kind:
        raise ValueError(f"{what}: another type than the operator's ({t.dtype})")
    return t.data_ptr(), stride[0], stride[1], n[1]


def _ints(t, shape, what: str):
    return _vec(t, shape, "torch.int32", what)


# ---- rotary positions ----------------------------------------------------------------------------------------------------
class Rotary:
    """How positions turn the first `rotated` values of a head (tsa_rotary_params)."""

    def __init__(self, rotated: int, *, base=10000.0, interleaved=False, factor=1.0, trained=0, low=1.0, high=4.0, amplitude=1.0):
        self.s = TsaRotary()
        _ok(_attn().tsa_rotary_init(TsaRotaryParams(base, factor, trained, low, high, amplitude, rotated, interleaved), self.s))


def rotate(rotary: Rotary, positions, q, k=None, q_out=None, k_out=None, *, backward=False, stream=None) -> None:
    """q, and k if there is one, turned by positions int32 [tokens] (tsa_rotate): in place, or to q_out and k_out. backward: the gradients of
    what was turned become those of what it was made from."""
    if k is None and k_out is not None:
        raise ValueError("k_out without k")
    kind, (tokens, _, dim) = _type(q), _three(q, "q")
    a = TsaRotateArgs(positions=_ints(positions, (tokens,), "positions"), tokens=tokens, head_dim=dim, type=kind, backward=backward)
    a.x[0] = _heads(q, "q")
    a.y[0] = a.x[0] if q_out is None else _heads(q_out, "q_out", q.shape, kind)
    if k is not None:
        a.x[1] = _heads(k, "k", (tokens, _three(k, "k")[1], dim), kind)
        a.y[1] = a.x[1] if k_out is None else _heads(k_out, "k_out", k.shape, kind)
    _same_device("rotate", positions, q, k, q_out, k_out)
    _ok(_attn().tsa_rotate(rotary.s, a, stream))


# ---- the cache -----------------------------------------------------------------------------------------------------------
def page_bytes(head_dim: int) -> int:
    """Bytes of a page of one head."""
    return 72 * head_dim


class Cache:
    """Pages of 4-bit keys and values: uint8 [n_pages][kv_heads][page_bytes(head_dim)], contiguous. Nothing has to be cleared."""

    def __init__(self, pages, kv_heads: int, head_dim: int):
        n = pages.shape[0]
        p = _vec(pages, (n, kv_heads, page_bytes(head_dim)), "torch.uint8", "pages")
        self.pages, self.s = pages, TsaCache(p, n, kv_heads, head_dim)


def _table(table):
    if len(table.shape) != 2 or str(table.dtype) != "torch.int32" or (table.shape[1] > 1 and table.stride()[1] != 1):
        raise ValueError(f"table: int32 [requests][pages] with contiguous rows, not {table.dtype} {tuple(table.shape)}")
    _device(table, "table")
    return table.data_ptr(), table.stride()[0]


def plan(lengths, fresh, table, free, n_free, first, positions, slots, status, *, ends=None, left=None, stream=None) -> None:
    """Pages, positions and slots of a step (tsa_cache_plan), all int32: lengths, fresh [requests], table [requests][pages], free [pages],
    n_free [1], first [requests + 1], positions and slots [rows], status [1]. ends and left None: lengths and n_free become them."""
    ends, left = lengths if ends is None else ends, n_free if left is None else left
    n, rows = lengths.shape[0], positions.shape[0]
    t, stride = _table(table)
    if table.shape[0] != n:
        raise ValueError(f"table: a row for each of {n} requests, not {table.shape[0]}")
    a = TsaCachePlanArgs(_ints(lengths, (n,), "lengths"), _ints(fresh, (n,), "fresh"), t, stride, _ints(free, (free.shape[0],), "free"),
                         _ints(n_free, (1,), "n_free"), _ints(ends, (n,), "ends"), _ints(left, (1,), "left"), _ints(first, (n + 1,), "first"),
                         _ints(positions, (rows,), "positions"), _ints(slots, (rows,), "slots"), _ints(status, (1,), "status"), n, table.shape[1],
                         free.shape[0], rows)
    _same_device("plan", lengths, fresh, table, free, n_free, first, positions, slots, status, ends, left)
    _ok(_attn().tsa_cache_plan(a, stream))


def slots(table, ends, first, positions, out, *, stream=None) -> None:
    """Positions and slots (out) of the rows first[i]..first[i + 1], the last tokens of request i's ends[i] (tsa_cache_slots)."""
    n, rows = ends.shape[0], positions.shape[0]
    t, stride = _table(table)
    if table.shape[0] != n:
        raise ValueError(f"table: a row for each of {n} requests, not {table.shape[0]}")
    a = TsaCachePlanArgs(table=t, table_stride=stride, ends=_ints(ends, (n,), "ends"), first=_ints(first, (n + 1,), "first"),
                         positions=_ints(positions, (rows,), "positions"), slots=_ints(out, (rows,), "slots"), requests=n, width=table.shape[1], rows=rows)
    _same_device("slots", table, ends, first, positions, out)
    _ok(_attn().tsa_cache_slots(a, stream))


def _rows(cache: Cache, k, v, slots, what: str):
    kind, tokens = _type(k), _three(k, "k")[0]
    shape = (tokens, cache.s.kv_heads, cache.s.head_dim)
    a = TsaCacheRowsArgs(_heads(k, "k", shape), _heads(v, "v", shape, kind), _ints(slots, (tokens,), "slots"), tokens, kind)
    _same_device(what, cache.pages, k, v, slots)
    return a


def store(cache: Cache, k, v, slots, *, stream=None) -> None:
    """Keys and values [tokens][kv_heads][head_dim] to slots int32 [tokens] as 4-bit values (tsa_cache_store)."""
    _ok(_attn().tsa_cache_store(cache.s, _rows(cache, k, v, slots, "store"), stream))


def load(cache: Cache, slots, k, v, *, stream=None) -> None:
    """What the slots hold to k and v (tsa_cache_load)."""
    _ok(_attn().tsa_cache_load(cache.s, _rows(cache, k, v, slots, "load"), stream))


def attend_cached_workspace(cache: Cache, q, table) -> int:
    """Workspace bytes of attend_cached; grows with q's rows and the table's requests and width."""
    a = TsaAttendCachedArgs(tokens=q.shape[0], requests=table.shape[0], width=table.shape[1], type=_type(q))
    a.q.heads = q.shape[1]
    return _attn().tsa_attend_cached_workspace(cache.s, a)


def attend_cached(cache: Cache, q, out, table, ends, first, *, scale=None, workspace=None, stream=None) -> None:
    """out = softmax(q K^T scale) V over the pages of each row's request (tsa_attend_cached). scale None: head_dim^-0.5."""
    kind, (tokens, _, dim), n = _type(q), _three(q, "q"), ends.shape[0]
    if dim != cache.s.head_dim:
        raise ValueError(f"q: heads of the cache's {cache.s.head_dim} values, not {dim}")
    t, stride = _table(table)
    if table.shape[0] != n:
        raise ValueError(f"table: a row for each of {n} requests, not {table.shape[0]}")
    a = TsaAttendCachedArgs(_heads(q, "q"), _heads(out, "out", q.shape, kind), t, stride, _ints(ends, (n,), "ends"),
                            _ints(first, (n + 1,), "first"), tokens, n, table.shape[1], kind, dim ** -0.5 if scale is None else scale)
    _same_device("attend_cached", cache.pages, q, out, table, ends, first, workspace)
    ws, size = _room(workspace)
    _ok(_attn().tsa_attend_cached(cache.s, a, ws, size, stream))


# ---- packed sequences ----------------------------------------------------------------------------------------------------
def _attend_args(q, k, v, out, lse, first, k_first, causal, scale):
    kind, (tokens, heads, dim), (k_tokens, kept) = _type(q), _three(q, "q"), _three(k, "k")[:2]
    n = 1 if first is None else first.shape[0] - 1
    return TsaAttendArgs(_heads(q, "q"), _heads(k, "k", (k_tokens, kept, dim), kind), _heads(v, "v", (k_tokens, kept, dim), kind),
                         _heads(out, "out", q.shape, kind), _ints(first, (n + 1,), "first"), _ints(k_first, (n + 1,), "k_first"),
                         _vec(lse, (heads, tokens), "torch.float32", "lse"), tokens, k_tokens, n, dim, kind, causal,
                         dim ** -0.5 if scale is None else scale)


def attend(q, k, v, out, *, lse=None, first=None, k_first=None, causal=True, scale=None, stream=None) -> None:
    """out = softmax(q K^T scale) V over packed sequences (tsa_attend); lse: float32 [heads][tokens]; first, k_first: int32
    [sequences + 1] (None: one sequence). scale None: head_dim^-0.5."""
    a = _attend_args(q, k, v, out, lse, first, k_first, causal, scale)
    _same_device("attend", q, k, v, out, lse, first, k_first)
    _ok(_attn().tsa_attend(a, stream))


def attend_backward_workspace(q, k) -> int:
    """Workspace bytes of attend_backward; grows with the rows."""
    a = TsaAttendArgs(tokens=q.shape[0], k_tokens=k.shape[0], sequences=1, head_dim=q.shape[2], type=_type(q))
    a.q.heads, a.k.heads, a.v.heads = q.shape[1], k.shape[1], k.shape[1]
    return _attn().tsa_attend_backward_workspace(a)


def attend_backward(q, k, v, out, dout, lse, dq=None, dk=None, dv=None, *, first=None, k_first=None, causal=True, scale=None,
                    workspace=None, stream=None) -> None:
    """The gradients of attend for dout that are asked for (tsa_attend_backward), from its inputs, out and lse."""
    g = TsaAttendGradArgs(_attend_args(q, k, v, out, lse, first, k_first, causal, scale))
    kind = g.f.type
    g.dout = _heads(dout, "dout", q.shape, kind)
    if dq is not None:
        g.dq = _heads(dq, "dq", q.shape, kind)
    if dk is not None:
        g.dk = _heads(dk, "dk", k.shape, kind)
    if dv is not None:
        g.dv = _heads(dv, "dv", v.shape, kind)
    _same_device("attend_backward", q, k, v, out, dout, lse, dq, dk, dv, first, k_first, workspace)
    ws, size = _room(workspace)
    _ok(_attn().tsa_attend_backward(g, ws, size, stream))
